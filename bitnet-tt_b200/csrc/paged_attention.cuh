// Attention of each sequence's new tokens over its paged keys and values.
//
// Sequence b has n = cu[b + 1] - cu[b] new tokens (packed rows of q) and
// kv_lens[b] keys, the new tokens' own among them.  Token i sees the keys
// j < kv_lens[b] - n + i + 1; a token that sees none gets zeros.
//     o = sum_j p_j v_j / sum_j p_j,   p_j = exp2(log2(e) scale q . k_j - m)
// with the running maximum m and the sum in fp32.
//
// The G = n_heads / n_kv query heads of a KV head share its keys, so a block of
// work is a run of packed rows of one (sequence, KV head): row r is token r / G,
// head g G + r % G.  Calls whose sequences have up to 32 rows (decode, a few drafted
// tokens) go to paged_rows_kernel here; in others the sequences of up to 8 rows (16 if
// G > 8) do, and longer ones go to paged_chunk_kernel (paged_chunk.cuh).  Both hold the
// weights of a sequence of up to 32 rows in 16 bits (bf16 caches), so its precision
// does not depend on what it is batched with.
#pragma once
#include <climits>

#include "attention.cuh"
#include "common.cuh"
#include "paged_kv.cuh"

namespace bitnet {

constexpr int PAGED_FINE = 32;  // rows of the longest sequence whose weights are held in 16 bits

// One block of rows: rows row0 .. row0 + nrows - 1 of sequence b.
struct PagedBlock {
  int b, row0, nrows;
  int tok0;    // the sequence's first packed token
  int past;    // kv_len - n: keys before the new tokens (may be negative)
  int kend;    // keys that the block's last row sees, not below 0
};

struct PagedAttnParams {
  PagedKV kv;
  const int32_t* cu;
  const int32_t* kv_lens;
  int B, tokens, max_q, max_kv;
  const uint16_t* q;
  int ld_q, n_heads, G;
  float scale_log2;    // scale * log2(e)
  int nsplit, span;    // the keys are cut into nsplit parts of span keys
  int blocks;          // grid.x: row blocks, an upper bound
  int small;           // chunk kernel: sequences of up to this many rows are not its own
  int most, per;       // rows kernel: rows of its longest sequences, and blocks of each
  int beside;          // rows kernel: launched after the chunk kernel, to run beside it
  float2* part_ml;     // [nsplit][blocks][n_kv][R] (maximum, sum)
  float* part_o;       // [nsplit][blocks][n_kv][R][D], unnormalised
  PagedBlock* found;   // chunk kernel with nsplit > 1: [blocks], nrows 0 where there is none
  uint16_t* out;       // [tokens][n_heads * D]
};

// Rows row0 .. of sequence b, which has n new tokens from packed row lo on and kv
// keys, in a block of up to R rows.  False when there are none, or when the
// lengths do not hold.
template <int R>
__device__ __forceinline__ bool paged_block_of(const PagedAttnParams& p, int b, int lo, int n, int kv, int row0, int lane,
                                               PagedBlock& o) {
  if (n == 0) return false;
  if (n < 0 || n > p.max_q || lo < 0 || lo > p.tokens - n || kv < 0 || kv > p.max_kv) {
    if (lane == 0) record_error(DEV_ERR_BOUNDS, 350);
    return false;
  }
  if (row0 >= n * p.G) return false;
  o.b = b;
  o.row0 = row0;
  o.nrows = min(R, n * p.G - row0);
  o.tok0 = lo;
  o.past = kv - n;
  o.kend = max(0, o.past + (row0 + o.nrows - 1) / p.G + 1);
  return true;
}

// Blocks of sequences of up to p.most rows, p.per blocks a sequence; the others
// are not this kernel's.
template <int R>
__device__ __forceinline__ bool paged_block_direct(const PagedAttnParams& p, int bx, int lane, PagedBlock& o) {
  const int b = bx / p.per, row0 = (bx - b * p.per) * R;
  const int lo = p.cu[b], n = p.cu[b + 1] - lo;
  if ((long long)n * p.G > p.most && (long long)p.max_q * p.G > p.most) return false;
  return paged_block_of<R>(p, b, lo, n, p.kv_lens[b], row0, lane, o);
}

// The R-row blocks of all sequences of more than p.small rows, numbered so that
// those with more keys come first (CTAs start in that order, so the long ones do
// not end last); whole warp.  Blocks are ranked by their 128-key tiles: the rank
// of block bx is found by bisection over the number of tiles, counting the blocks
// with at least that many by arithmetic (a sequence's later blocks see more).
// Equal ranks are in the order of sequences.  Up to 128 sequences; beyond that the
// blocks are in the order of sequences alone, the last first.
// C: sequences of a lane; cold code, so the common case has its own shorter copy.
template <int R, int C>
__device__ __forceinline__ bool paged_block_ranked(const PagedAttnParams& p, int bx, int lane, PagedBlock& o) {
  int at[C], len[C], kv[C], rows[C], past[C], nb = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int b = 32 * c + lane;
    at[c] = len[c] = kv[c] = rows[c] = past[c] = 0;
    if (b < p.B) {
      at[c] = p.cu[b];
      len[c] = p.cu[b + 1] - at[c];
      kv[c] = p.kv_lens[b];
      const int n = min(max(len[c], 0), p.max_q);
      past[c] = min(kv[c], p.max_kv) - n;
      rows[c] = n * p.G > p.small ? n * p.G : 0;
      if (len[c] < 0) rows[c] = 1, past[c] = -1;  // a block that reports it, behind all others
      nb += (rows[c] + R - 1) / R;
    }
  }
  // the blocks of at least t tiles of sequence c: those whose last row's token is y or later
  auto count = [&](int c, int t) {
    const int all = (rows[c] + R - 1) / R;
    const long long y = (long long)(t - 1) * 128 - past[c];
    if (t <= 0 || y <= 0 || all == 0) return all;
    const long long first = y * p.G;  // the first row of token y
    return first >= rows[c] ? 0 : all - (int)(first / R);
  };
  auto total = [&](int t) {
    int n = 0;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (32 * c < p.B) n += count(c, t);
    return (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
  };
  if (bx >= (int)__reduce_add_sync(0xffffffffu, (unsigned)nb)) return false;
  int lo = 0, hi = (p.max_kv + 127) / 128 + 1;  // more than bx blocks have lo tiles, not more have hi
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (total(mid) > bx) lo = mid;
    else hi = mid;
  }
  // among the blocks of exactly lo tiles
  int rank = bx - total(lo + 1);
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (32 * c >= p.B) break;
    const int above = count(c, lo + 1), here = count(c, lo) - above;
    int sum = here;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    const unsigned over = __ballot_sync(0xffffffffu, sum > rank);
    if (over) {
      const int src = __ffs(over) - 1;
      rank -= __shfl_sync(0xffffffffu, sum - here, src);
      const int last = __shfl_sync(0xffffffffu, (rows[c] + R - 1) / R - 1 - above, src);
      return paged_block_of<R>(p, 32 * c + src, __shfl_sync(0xffffffffu, at[c], src), __shfl_sync(0xffffffffu, len[c], src),
                               __shfl_sync(0xffffffffu, kv[c], src), (last - rank) * R, lane, o);
    }
    rank -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}
template <int R>
__device__ __forceinline__ bool paged_block_search(const PagedAttnParams& p, int bx, int lane, PagedBlock& o) {
  if (p.B <= 32) return paged_block_ranked<R, 1>(p, bx, lane, o);
  if (p.B <= 128) return paged_block_ranked<R, 4>(p, bx, lane, o);
  bx = p.blocks - 1 - bx;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int i = b0 + lane;
    const int len = i < p.B ? p.cu[i + 1] - p.cu[i] : 0, rows = min(max(len, 0), p.max_q) * p.G;
    const int nb = len < 0 ? 1 : rows > p.small ? (rows + R - 1) / R : 0;
    int sum = nb;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    const unsigned above = __ballot_sync(0xffffffffu, sum > bx);
    if (above) {
      const int src = __ffs(above) - 1, b = b0 + src;
      return paged_block_of<R>(p, b, p.cu[b], p.cu[b + 1] - p.cu[b], p.kv_lens[b],
                               (bx - __shfl_sync(0xffffffffu, sum - nb, src)) * R, lane, o);
    }
    bx -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

__device__ __forceinline__ int paged_parts(const PagedAttnParams& p, int kend) {
  return max(1, (kend + p.span - 1) / p.span);
}

// ---------------------------------------------------------------------------
// few rows: mma.sync
// ---------------------------------------------------------------------------
// A CTA of 4 warps takes up to 8 H rows of one (sequence, KV head) over one part of
// the keys; warp w the tiles w, w + 4, ... of 16 keys (int8: 32).  K
// and V rows come by 16-byte cp.async into buffers of the warp's own, 16 KB in
// flight a warp, so no barrier is needed inside the loop.  Products run on
// m16n8k16 with fp32 sums: S = Q K^T, then for H = 1 (8 rows) O^T += V^T P^T, whose
// output columns are the 8 rows, for H = 2 O += P V.  As in paged_chunk.cuh the
// maximum is lazy: O and the sums are rescaled when it grew by more than 2^8.
// bf16 caches: P enters as a bf16 pair hi + lo (16 significant bits).
//
// int8: the kernel would be bound by the integer pipe, which turns codes into
// 16-bit floats, so it works in f16, where that costs three operations for four
// codes: (w & 0x00FF00FF) ^ 0x64806480 holds 1152 + code twice, and subtracting
// 1152 is exact (and runs elsewhere).  The bf16 form cost five and two; 256
// ragged sequences of up to 4K keys took 256 us with it, 143 now (4.8 TB/s).
//  * Q in f16: scaled by a power of two per row so that its largest value is
//    2^13 .. 2^14, which keeps every bit of elements down to 2^-27 of it.
//  * P in f16, 11 significant bits.  The values' scales vs_j can differ by any
//    factor, so the weights p_j vs_j have a running maximum of their own: they are
//    exp2(x_j + log2 vs_j - mv + 7) next to the sum's exp2(x_j - m).  With the 7
//    the largest weight lies in 2^7 .. 2^15, and the step of the smallest f16, 2^-24,
//    is below 2^-31 of it.
//  * Dims of S and output columns of O are permuted so that each thread's bytes
//    are what its fragments need.
constexpr int PRA_WARPS = 4;
constexpr int PRA_THREADS = PRA_WARPS * 32;
constexpr float PRA_GROWTH = 8.f;
constexpr float PRA_LIFT = 7.f;

template <int D, bool I8, int H>
struct PraShape {
  static constexpr int R = 8 * H;                        // rows
  static constexpr int KT = I8 ? 32 : 16;                // keys of a tile
  static constexpr int ROW = D * (I8 ? 1 : 2);           // bytes of a row
  static constexpr int CPR = ROW / 16;                   // 16-byte chunks of a row
  static constexpr int HALF = KT * ROW;                  // K (or V) of a tile
  static constexpr int BUF = 2 * HALF + (I8 ? 256 : 0);  // + 32 key and 32 value scales
  static constexpr int NBUF = 8192 / HALF;
  static constexpr int SMEM_TILES = PRA_WARPS * NBUF * BUF;
  static constexpr int SMEM_MERGE = PRA_WARPS * R * (D + 2) * 4;
  static constexpr int SMEM = SMEM_TILES > SMEM_MERGE ? SMEM_TILES : SMEM_MERGE;
};

// Byte offset of chunk c of row r.  The chunk is moved within its row so that
// the rows one access reads at the same chunk fall in different banks: 8 rows
// for ldmatrix, and for the int8 keys two rows' halves.
template <int CPR, bool KEYS8>
__device__ __forceinline__ uint32_t pra_off(int r, int c) {
  if (KEYS8 && CPR == 8) return (uint32_t)(r * 128 + ((c ^ ((r & 1) << 2)) << 4));
  if (CPR == 4) return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
  return (uint32_t)(r * CPR * 16 + ((c ^ (r & 7)) << 4));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// the codes in bytes 0 and 2 of w as an f16 pair
__device__ __forceinline__ uint32_t codes_f2(uint32_t w) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"((w & 0x00FF00FFu) ^ 0x64806480u), "r"(0x64806480u));
  return d;
}
__device__ __forceinline__ uint32_t f16x2_of(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <bool F16>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4_zfill(uint32_t dst, const void* src, uint32_t src_bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// two values as a bf16 pair, and what that leaves as another
__device__ __forceinline__ void split_bf2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = bf2_of(a, b);
  lo = bf2_of(__fsub_rn(a, __uint_as_float(hi << 16)), __fsub_rn(b, __uint_as_float(hi & 0xFFFF0000u)));
}
// The maximum of a running softmax after one more tile, and the factor that
// what was summed under the old one takes (1 while it stays).
__device__ __forceinline__ float pra_grow(float& m, float top) {
  const float mn = fmaxf(m, top);
  const float f = mn == -INFINITY ? 1.f : ex2(m - mn);
  m = mn;
  return f;
}

template <int D, bool I8, int H>
__global__ void __launch_bounds__(PRA_THREADS, 3) paged_rows_kernel(const PagedAttnParams p) {
  using S = PraShape<D, I8, H>;
  constexpr int KT = S::KT, NT = KT / 8;  // n-tiles of 8 keys
  extern __shared__ __align__(128) uint8_t smem_pra[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  const int g = blockIdx.y, sp = blockIdx.z;
  // Beside the chunk kernel there is nothing to wait for: its CTAs wait for what came before, and the
  // first one fences, ahead of the triggers that allow this launch.  A trigger publishes nothing, so this
  // side fences too: whatever stands in this SM's L1 from before is dropped, and the loads below
  // find in L2 what the chunk kernel's wait made visible.  (With a wait for the chunk kernel instead, 3
  // chunks of 1024 beside 45 int8 decode rows take 148 us for 133, 4 of 256 beside 60 in bf16 76 for 48.)
  // The last CTA waits for the chunk kernel before it ends, so that what follows this kernel follows both.
  if (p.beside) fence_acq_rel_gpu();
  else pdl_wait();
  const bool closes = p.beside && blockIdx.x == gridDim.x - 1 && g == (int)gridDim.y - 1 && sp == (int)gridDim.z - 1;
  PagedBlock blk;
  const bool found = paged_block_direct<S::R>(p, blockIdx.x, lane, blk);
  const int nparts = found ? paged_parts(p, blk.kend) : 0;
  if (sp >= nparts) {
    if (closes) pdl_wait();
    return;
  }
  const int k0 = sp * p.span, k1 = min(blk.kend, k0 + p.span);  // this part's keys
  const int ntiles = max(0, (k1 - k0 + KT - 1) / KT);
  const int ntw = ntiles > warp ? (ntiles - warp + PRA_WARPS - 1) / PRA_WARPS : 0;
  const uint32_t buf0 = smem_u32(smem_pra) + warp * S::NBUF * S::BUF;
  const int32_t* table = p.kv.table + (size_t)blk.b * p.kv.max_pages;
  const int slot_mask = (1 << p.kv.page_shift) - 1;

  constexpr int HT = KT / 16;  // 16-key pieces of a tile: each lies in one page
  int pages = -1;              // lane l: the page of piece l % HT of this warp's tile (i / (32 / HT)) * (32 / HT) + l / HT
  auto issue = [&](int i) {
    if (i % (32 / HT) == 0) {
      const int t0 = k0 + (warp + (i + lane / HT) * PRA_WARPS) * KT + (lane % HT) * 16;
      pages = -1;
      if (t0 < k1) {
        pages = table[t0 >> p.kv.page_shift];
        if (pages < 0 || pages >= p.kv.num_pages) {
          record_error(DEV_ERR_BOUNDS, 351);
          pages = -1;
        }
      }
    }
    const int t0 = k0 + (warp + i * PRA_WARPS) * KT;
    const uint32_t base = buf0 + (i % S::NBUF) * S::BUF;
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      const int page = __shfl_sync(0xffffffffu, pages, (i % (32 / HT)) * HT + ht);
      const int nk = page < 0 ? 0 : k1 - t0 - 16 * ht;  // live rows, 16 or more: all
      const size_t row0 = paged_row(p.kv, max(page, 0), g, (t0 + 16 * ht) & slot_mask);
      // chunk lane % CPR of the rows lane / CPR + k * (32 / CPR): the addresses of the
      // copies differ by constants (the swizzle repeats every 8 rows)
      const uint8_t* src_k = p.kv.k + row0 * S::ROW + lane * 16;
      const uint8_t* src_v = p.kv.v + row0 * S::ROW + lane * 16;
      constexpr int RPC = 32 / S::CPR;  // rows of one copy instruction
#pragma unroll
      for (int k = 0; k < S::CPR / 2; ++k) {
        const int row = lane / S::CPR + k * RPC, c = lane % S::CPR;
        constexpr int REP = RPC >= 8 ? 1 : 8 / RPC;
        const int low = lane / S::CPR + (k % REP) * RPC;  // row % 8
        const uint32_t rest = (16 * ht + (k / REP) * REP * RPC) * S::ROW;
        const uint32_t at_k = base + pra_off<S::CPR, I8>(low, c) + rest;
        const uint32_t at_v = base + S::HALF + pra_off<S::CPR, false>(low, c) + rest;
        if (nk >= 16) {
          cp_async16(at_k, src_k + k * 512);
          cp_async16(at_v, src_v + k * 512);
        } else {
          const uint32_t bytes = row < nk ? 16u : 0u;
          cp_async16_zfill(at_k, bytes ? src_k + k * 512 : p.kv.k, bytes);
          cp_async16_zfill(at_v, bytes ? src_v + k * 512 : p.kv.v, bytes);
        }
      }
      if (I8) {
        const int row = lane & 15;
        const float* src = (lane < 16 ? p.kv.ks : p.kv.vs) + row0 + (row < nk ? row : 0);
        cp_async4_zfill(base + 2 * S::HALF + (lane >> 4) * 128 + (16 * ht + row) * 4, src, row < nk ? 4u : 0u);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < S::NBUF; ++i) {
    if (i < ntw) issue(i);
    cp_async_commit();
  }

  // query fragments of rows qr (and qr + 8)
  const int qr = lane >> 2, qc = lane & 3;
  uint32_t qa[D / 16][2 * H];  // [.][h]: the first pair, [.][H + h]: the second
  int lim[H];                  // keys that the rows see
  float fac[H];                // scale * log2(e), for int8 with Q's power of two taken out
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int r = blk.row0 + qr + 8 * h;
    const bool in = qr + 8 * h < blk.nrows;
    const int tok = r / p.G, head = g * p.G + r - tok * p.G;
    lim[h] = in ? blk.past + tok + 1 : INT_MAX;
    fac[h] = p.scale_log2;
    const uint16_t* row = p.q + (size_t)(blk.tok0 + (in ? tok : 0)) * p.ld_q + (in ? head : 0) * D;
    if (I8) {
      // dims 64 (ks / 4) + 16 qc + 4 (ks % 4) + e: e = 0, 2 in the first pair, 1, 3 in the second
      uint2 w[D / 16];
      uint32_t top = 0;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        w[ks] = make_uint2(0, 0);
        if (in) w[ks] = *reinterpret_cast<const uint2*>(row + 64 * (ks / 4) + 16 * qc + 4 * (ks % 4));
        top = max(max(top, w[ks].x & 0x7fffu), (w[ks].x >> 16) & 0x7fffu);
        top = max(max(top, w[ks].y & 0x7fffu), (w[ks].y >> 16) & 0x7fffu);
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t up = 267u - max(top >> 7, 20u);  // exponent field of 2^13 / 2^floor(log2 max)
      const float f = __uint_as_float(up << 23);
      fac[h] *= __uint_as_float((254u - up) << 23);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const float e0 = __uint_as_float(w[ks].x << 16), e1 = __uint_as_float(w[ks].x & 0xFFFF0000u);
        const float e2 = __uint_as_float(w[ks].y << 16), e3 = __uint_as_float(w[ks].y & 0xFFFF0000u);
        qa[ks][h] = f16x2_of(e0 * f, e2 * f);
        qa[ks][H + h] = f16x2_of(e1 * f, e3 * f);
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qa[ks][h] = in ? *reinterpret_cast<const uint32_t*>(row + 16 * ks + 2 * qc) : 0u;
        qa[ks][H + h] = in ? *reinterpret_cast<const uint32_t*>(row + 16 * ks + 8 + 2 * qc) : 0u;
      }
    }
  }
  const int lim_lo = blk.past + blk.row0 / p.G + 1;  // the first row's: it sees the fewest
  float m[H], l[H], mv[H];  // maximum and this lane's share of the sum; maximum of the weights (int8)
#pragma unroll
  for (int h = 0; h < H; ++h) m[h] = mv[h] = -INFINITY, l[h] = 0.f;
  // H = 1: O^T, m-tile j = dims, columns = rows 2 qc, + 1.  H = 2: O, n-tile j = dims, rows qr, qr + 8.
  constexpr int NO = H == 1 ? D / 16 : D / 8;
  float o[NO][4];
#pragma unroll
  for (int j = 0; j < NO; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
  const int mi = lane >> 3, mr = lane & 7;

  for (int i = 0; i < ntw; ++i) {
    cp_async_wait<S::NBUF - 1>();
    __syncwarp();
    const uint32_t kb = buf0 + (i % S::NBUF) * S::BUF, vb = kb + S::HALF;
    const int t0 = k0 + (warp + i * PRA_WARPS) * KT;
    float s[NT][4];  // keys 8 n + 2 qc, + 1 of rows qr (0, 1) and qr + 8 (2, 3)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
    auto qk = [&](float(&d)[4], int ks, uint32_t b0, uint32_t b1) {
      mma_16816<I8>(d, qa[ks][0], H == 2 ? qa[ks][1] : 0u, qa[ks][H], H == 2 ? qa[ks][H + H - 1] : 0u, b0, b1);
    };
    if (I8) {
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t w[4];
          const uint32_t a = kb + pra_off<S::CPR, true>(8 * n + qr, 4 * h + qc);
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
#pragma unroll
          for (int k = 0; k < 4; ++k) qk(s[n], 4 * h + k, codes_f2(w[k]), codes_f2(w[k] >> 8));
        }
    } else {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4(kb + pra_off<S::CPR, false>((mi >> 1) * 8 + mr, 2 * ks + (mi & 1)), b0, b1, b2, b3);
        qk(s[0], ks, b0, b1);
        qk(s[1], ks, b2, b3);
      }
    }
    // scores in base 2; v: log2 of the values' scales
    const bool masked = t0 + KT > min(lim_lo, k1);
    float2 v[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float2 k;
      if (I8) {
        const uint32_t a = kb + 2 * S::HALF + (8 * n + 2 * qc) * 4;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(k.x), "=f"(k.y) : "r"(a));
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v[n].x), "=f"(v[n].y) : "r"(a + 128));
        v[n].x = lg2(v[n].x), v[n].y = lg2(v[n].y);
      }
#pragma unroll
      for (int e = 0; e < 2 * H; ++e) {
        s[n][e] *= fac[e >> 1];
        if (I8) s[n][e] *= (e & 1) ? k.y : k.x;
      }
    }
    auto hidden = [&](int n, int e) { return t0 + 8 * n + 2 * qc + (e & 1) >= min(lim[e >> 1], k1); };
    if (masked) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2 * H; ++e)
          if (hidden(n, e)) s[n][e] = -INFINITY;
    }
    // int8: a hidden key's value scale may be anything, so its maximum (a NaN is passed over) only
    // sets a reference, and its weight is cleared below
    float top[H], topv[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      top[h] = topv[h] = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        top[h] = fmaxf(fmaxf(top[h], s[n][2 * h]), s[n][2 * h + 1]);
        if (I8) topv[h] = fmaxf(fmaxf(topv[h], s[n][2 * h] + v[n].x), s[n][2 * h + 1] + v[n].y);
      }
    }
    bool grown = false;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      grown = grown || top[h] > m[h] + PRA_GROWTH;
      if (I8) {
        topv[h] = fmaxf(topv[h], __shfl_xor_sync(0xffffffffu, topv[h], 1));
        topv[h] = fmaxf(topv[h], __shfl_xor_sync(0xffffffffu, topv[h], 2));
        grown = grown || topv[h] > mv[h] + PRA_GROWTH;
      }
    }
    if (__any_sync(0xffffffffu, grown)) {
      float f[H];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        f[h] = pra_grow(m[h], top[h]);
        l[h] *= f[h];
        if (I8) f[h] = pra_grow(mv[h], topv[h]);
      }
      if (H == 1) {  // the states of rows 2 qc and 2 qc + 1 are in lanes 8 qc and 8 qc + 4
        const float lo = __shfl_sync(0xffffffffu, f[0], 8 * qc), hi = __shfl_sync(0xffffffffu, f[0], 8 * qc + 4);
#pragma unroll
        for (int j = 0; j < NO; ++j) o[j][0] *= lo, o[j][1] *= hi, o[j][2] *= lo, o[j][3] *= hi;
      } else {
#pragma unroll
        for (int j = 0; j < NO; ++j) o[j][0] *= f[0], o[j][1] *= f[0], o[j][2] *= f[H - 1], o[j][3] *= f[H - 1];
      }
    }
    float ref[H], refv[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      ref[h] = m[h] == -INFINITY ? 0.f : m[h];  // a row that has seen no key yet
      refv[h] = mv[h] == -INFINITY ? 0.f : mv[h] - PRA_LIFT;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2 * H; ++e) {
        const int h = e >> 1;
        const float x = s[n][e], w = ex2(x - ref[h]);
        l[h] += w;
        s[n][e] = I8 ? ex2(x + ((e & 1) ? v[n].y : v[n].x) - refv[h]) : w;
      }
    if (I8 && masked) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2 * H; ++e)
          if (hidden(n, e)) s[n][e] = 0.f;
    }
#pragma unroll
    for (int kk = 0; kk < KT / 16; ++kk) {  // 16 keys
      // rows qr: keys 2 qc, + 1 of the first and the second 8; then rows qr + 8
      uint32_t ph[2 * H], pl[2 * H];
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float a = s[2 * kk + n][2 * h], b = s[2 * kk + n][2 * h + 1];
          if (I8) ph[2 * h + n] = f16x2_of(a, b);
          else split_bf2(a, b, ph[2 * h + n], pl[2 * h + n]);
        }
      // O += (rows) P V, or O^T with V^T as the left operand
      auto pv = [&](float(&d)[4], uint32_t v0, uint32_t v1, const uint32_t(&w)[2 * H]) {
        mma_16816<I8>(d, w[0], H == 2 ? w[H] : 0u, w[1], H == 2 ? w[H + 1] : 0u, v0, v1);
      };
      const int key = 16 * kk;
      if (I8) {
#pragma unroll
        for (int jj = 0; jj < S::CPR / 2; ++jj) {
          // transposed 8 x 8 pairs of bytes: (keys 0-7, chunk 2 jj), (8-15, 2 jj), (0-7, 2 jj + 1), (8-15, 2 jj + 1)
          uint32_t x[4];
          ldsm_x4_t(vb + pra_off<S::CPR, false>(key + (mi & 1) * 8 + mr, 2 * jj + (mi >> 1)), x[0], x[1], x[2], x[3]);
#pragma unroll
          for (int c = 0; c < 2; ++c) {  // a chunk holds 16 dims: even ones, odd ones
            const uint32_t e0 = codes_f2(x[2 * c]), o0 = codes_f2(x[2 * c] >> 8);
            const uint32_t e1 = codes_f2(x[2 * c + 1]), o1 = codes_f2(x[2 * c + 1] >> 8);
            if (H == 1) {
              mma_16816<I8>(o[2 * jj + c], e0, o0, e1, o1, ph[0], ph[1]);
            } else {
              pv(o[(4 * jj + 2 * c) % NO], e0, e1, ph);
              pv(o[(4 * jj + 2 * c + 1) % NO], o0, o1, ph);
            }
          }
        }
      } else {
#pragma unroll
        for (int jj = 0; jj < S::CPR / 2; ++jj) {
          uint32_t a0, a1, a2, a3;
          if (H == 1) {
            // (keys 0-7, chunk 2 jj), (0-7, 2 jj + 1), (8-15, 2 jj), (8-15, 2 jj + 1)
            ldsm_x4_t(vb + pra_off<S::CPR, false>(key + (mi >> 1) * 8 + mr, 2 * jj + (mi & 1)), a0, a1, a2, a3);
            mma_16816<I8>(o[jj], a0, a1, a2, a3, ph[0], ph[1]);
            mma_16816<I8>(o[jj], a0, a1, a2, a3, pl[0], pl[1]);
          } else {
            // (keys 0-7, chunk 2 jj), (8-15, 2 jj), (0-7, 2 jj + 1), (8-15, 2 jj + 1)
            ldsm_x4_t(vb + pra_off<S::CPR, false>(key + (mi & 1) * 8 + mr, 2 * jj + (mi >> 1)), a0, a1, a2, a3);
            pv(o[(2 * jj) % NO], a0, a1, ph);
            pv(o[(2 * jj + 1) % NO], a2, a3, ph);
            pv(o[(2 * jj) % NO], a0, a1, pl);
            pv(o[(2 * jj + 1) % NO], a2, a3, pl);
          }
        }
      }
    }
    __syncwarp();
    if (i + S::NBUF < ntw) issue(i + S::NBUF);
    cp_async_commit();
  }
  cp_async_wait<0>();
  __syncthreads();  // the tiles' memory is free

  // the warps' states: [warp][row] (m, l), then [warp][row][D], outputs under m
  float2* sm_ml = reinterpret_cast<float2*>(smem_pra);
  float* sm_o = reinterpret_cast<float*>(sm_ml + PRA_WARPS * S::R);
  float fv[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (qc == 0) sm_ml[warp * S::R + qr + 8 * h] = make_float2(m[h], l[h]);
    fv[h] = !I8 ? 1.f : (mv[h] == -INFINITY ? 0.f : ex2(mv[h] - PRA_LIFT - m[h]));
  }
  if (H == 1) {
    const float lo = __shfl_sync(0xffffffffu, fv[0], 8 * qc), hi = __shfl_sync(0xffffffffu, fv[0], 8 * qc + 4);
    float* d0 = sm_o + (size_t)(warp * S::R + 2 * qc) * D;
#pragma unroll
    for (int j = 0; j < NO; ++j) {
      const int a = I8 ? 16 * j + 2 * qr : 16 * j + qr, b = I8 ? a + 1 : a + 8;
      d0[a] = o[j][0] * lo;
      d0[D + a] = o[j][1] * hi;
      d0[b] = o[j][2] * lo;
      d0[D + b] = o[j][3] * hi;
    }
  } else {
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int j = 0; j < NO; ++j) {
        // int8: n-tile j holds the dims of parity j % 2 of chunk j / 2
        const int d = I8 ? 16 * (j >> 1) + 4 * qc + (j & 1) : 8 * j + 2 * qc;
        float* dst = sm_o + (size_t)(warp * S::R + qr + 8 * h) * D + d;
        dst[0] = o[j][2 * h] * fv[h];
        dst[I8 ? 2 : 1] = o[j][2 * h + 1] * fv[h];
      }
  }
  __syncthreads();
  const size_t pb = ((size_t)sp * p.blocks + blockIdx.x) * p.kv.n_kv + g;
  for (int idx = tid; idx < blk.nrows * (D / 4); idx += PRA_THREADS) {
    const int r = idx / (D / 4), d = (idx % (D / 4)) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < PRA_WARPS; ++w) M = fmaxf(M, sm_ml[w * S::R + r].x);
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
#pragma unroll
    for (int w = 0; w < PRA_WARPS; ++w) {
      const float2 ml = sm_ml[w * S::R + r];
      const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
      const float4 a = *reinterpret_cast<const float4*>(sm_o + (size_t)(w * S::R + r) * D + d);
      num.x = fmaf(a.x, f, num.x), num.y = fmaf(a.y, f, num.y);
      num.z = fmaf(a.z, f, num.z), num.w = fmaf(a.w, f, num.w);
      den = fmaf(ml.y, f, den);
    }
    if (nparts == 1) {
      const float inv = M == -INFINITY ? 0.f : 1.f / den;
      const int row = blk.row0 + r, tok = row / p.G;
      uint16_t* dst = p.out + ((size_t)(blk.tok0 + tok) * p.n_heads + g * p.G + row - tok * p.G) * D + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(bf2_of(num.x * inv, num.y * inv), bf2_of(num.z * inv, num.w * inv));
    } else {
      if (d == 0) p.part_ml[pb * S::R + r] = make_float2(M, den);
      *reinterpret_cast<float4*>(p.part_o + (pb * S::R + r) * D + d) = num;
    }
  }
  if (closes) pdl_wait();
}

// ---------------------------------------------------------------------------
// joining the parts
// ---------------------------------------------------------------------------
// Parts' unnormalised outputs are weighed by exp2(m_part - max).  A block whose
// keys fit in one part was written by its own CTA.  The rows kernel's: W warps a
// row, each the parts w, w + W, ..., so that with many parts the chain of loads is
// short.
template <int D, int R, int W>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedAttnParams p) {
  constexpr int V = D / 32;
  __shared__ float s_num[4][D], s_den[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = blockIdx.z * (4 / W) + warp / W, w = warp % W, g = blockIdx.y;
  pdl_trigger();
  pdl_wait();
  PagedBlock blk;
  if (!paged_block_direct<R>(p, blockIdx.x, lane, blk)) return;
  const int nparts = paged_parts(p, blk.kend);
  if (nparts == 1) return;
  const size_t step = (size_t)p.blocks * p.kv.n_kv;
  const size_t pb = (size_t)blockIdx.x * p.kv.n_kv + g;
  float num[V], den = 0.f, M = -INFINITY;
#pragma unroll
  for (int e = 0; e < V; ++e) num[e] = 0.f;
  if (r < blk.nrows) {
    for (int s = lane; s < nparts; s += 32) M = fmaxf(M, p.part_ml[(pb + s * step) * R + r].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
#pragma unroll 4
    for (int s = w; s < nparts; s += W) {
      const size_t at = (pb + s * step) * R + r;
      const float2 ml = p.part_ml[at];
      const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
      den = fmaf(ml.y, f, den);
#pragma unroll
      for (int e = 0; e < V; ++e) num[e] = fmaf(p.part_o[at * D + lane * V + e], f, num[e]);
    }
  }
  if (W > 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) s_num[warp][lane * V + e] = num[e];
    if (lane == 0) s_den[warp] = den;
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int x = 1; x < W; ++x) {
      den += s_den[warp + x];
#pragma unroll
      for (int e = 0; e < V; ++e) num[e] += s_num[warp + x][lane * V + e];
    }
  }
  if (r >= blk.nrows) return;
  const float inv = M == -INFINITY ? 0.f : 1.f / den;
  const int row = blk.row0 + r, tok = row / p.G;
  uint32_t* dst = reinterpret_cast<uint32_t*>(
      p.out + ((size_t)(blk.tok0 + tok) * p.n_heads + g * p.G + row - tok * p.G) * D + lane * V);
#pragma unroll
  for (int e = 0; e < V / 2; ++e) dst[e] = bf2_of(num[2 * e] * inv, num[2 * e + 1] * inv);
}

template <int V>
__device__ __forceinline__ void load_f(const float* src, float* x) {
  if constexpr (V == 4) {
    const float4 v = *reinterpret_cast<const float4*>(src);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const float2 v = *reinterpret_cast<const float2*>(src);
    x[0] = v.x, x[1] = v.y;
  }
}

// The chunk kernel's blocks of R rows in few parts: N rows a warp, whose loads do
// not wait for one another.  The blocks are as the chunk kernel found them (a
// search of its own in each of these short CTAs cost 80 us where the parts' bytes
// take 20).
constexpr int PJC_N = 4;
template <int D, int R>
__global__ void __launch_bounds__(128) paged_chunk_join_kernel(const PagedAttnParams p) {
  constexpr int V = D / 32, N = PJC_N;
  const int lane = threadIdx.x & 31, g = blockIdx.y;
  const int r0 = (blockIdx.z * 4 + (threadIdx.x >> 5)) * N;
  pdl_trigger();
  pdl_wait();
  const PagedBlock blk = p.found[blockIdx.x];
  if (r0 >= blk.nrows) return;
  const int nparts = paged_parts(p, blk.kend);
  if (nparts == 1) return;
  const size_t step = (size_t)p.blocks * p.kv.n_kv;
  const size_t pb = (size_t)blockIdx.x * p.kv.n_kv + g;
  float num[N][V], den[N], M[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    den[k] = 0.f;
    M[k] = -INFINITY;
#pragma unroll
    for (int e = 0; e < V; ++e) num[k][e] = 0.f;
  }
  // rows past the block's last read the last one's parts and are not stored
  for (int s = lane; s < nparts; s += 32)
#pragma unroll
    for (int k = 0; k < N; ++k) M[k] = fmaxf(M[k], p.part_ml[(pb + s * step) * R + min(r0 + k, blk.nrows - 1)].x);
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M[k] = fmaxf(M[k], __shfl_xor_sync(0xffffffffu, M[k], o));
#pragma unroll 2
  for (int s = 0; s < nparts; ++s) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const size_t at = (pb + s * step) * R + min(r0 + k, blk.nrows - 1);
      const float2 ml = p.part_ml[at];
      float x[V];
      load_f<V>(p.part_o + at * D + lane * V, x);
      const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - M[k]);
      den[k] = fmaf(ml.y, f, den[k]);
#pragma unroll
      for (int e = 0; e < V; ++e) num[k][e] = fmaf(x[e], f, num[k][e]);
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if (r0 + k >= blk.nrows) break;
    const float inv = M[k] == -INFINITY ? 0.f : 1.f / den[k];
    const int row = blk.row0 + r0 + k, tok = row / p.G;
    uint32_t* dst = reinterpret_cast<uint32_t*>(
        p.out + ((size_t)(blk.tok0 + tok) * p.n_heads + g * p.G + row - tok * p.G) * D + lane * V);
#pragma unroll
    for (int e = 0; e < V / 2; ++e) dst[e] = bf2_of(num[k][2 * e] * inv, num[k][2 * e + 1] * inv);
  }
}

}  // namespace bitnet
