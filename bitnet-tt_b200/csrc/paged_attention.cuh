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
// head g G + r % G.  Sequences of up to 16 rows (decode, a few drafted tokens) go to
// paged_rows_kernel here, longer ones to paged_chunk_kernel (paged_chunk.cuh).
#pragma once
#include "attention.cuh"
#include "common.cuh"
#include "paged_kv.cuh"

namespace bitnet {

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
  float2* part_ml;     // [nsplit][blocks][n_kv][R] (maximum, sum)
  float* part_o;       // [nsplit][blocks][n_kv][R][D], unnormalised
  uint16_t* out;       // [tokens][n_heads * D]
};

// One block of rows: rows row0 .. row0 + nrows - 1 of sequence b.
struct PagedBlock {
  int b, row0, nrows;
  int tok0;    // the sequence's first packed token
  int past;    // kv_len - n: keys before the new tokens (may be negative)
  int kend;    // keys that the block's last row sees, not below 0
};

// Rows row0 .. of sequence b in a block of up to R rows.  False when the sequence
// has no new token, or when its lengths do not hold.
template <int R>
__device__ __forceinline__ bool paged_block_of(const PagedAttnParams& p, int b, int row0, int lane, PagedBlock& o) {
  const int lo = p.cu[b], n = p.cu[b + 1] - lo, kv = p.kv_lens[b];
  if (n == 0) return false;
  if (n < 0 || n > p.max_q || lo < 0 || lo > p.tokens - n || kv < 0 || kv > p.max_kv) {
    if (lane == 0) record_error(DEV_ERR_BOUNDS, 350);
    return false;
  }
  o.b = b;
  o.row0 = row0;
  o.nrows = min(R, n * p.G - row0);
  o.tok0 = lo;
  o.past = kv - n;
  o.kend = max(0, o.past + (row0 + o.nrows - 1) / p.G + 1);
  return true;
}

// Sequences of up to R rows: block b is sequence b; the others are not this
// kernel's.
template <int R>
__device__ __forceinline__ bool paged_block_direct(const PagedAttnParams& p, int b, int lane, PagedBlock& o) {
  if ((long long)(p.cu[b + 1] - p.cu[b]) * p.G > R && p.max_q * p.G > R) return false;
  return paged_block_of<R>(p, b, 0, lane, o);
}

// Block bx of the R-row blocks of all sequences of more than p.small rows, in
// order; whole warp.
template <int R>
__device__ __forceinline__ bool paged_block_search(const PagedAttnParams& p, int bx, int lane, PagedBlock& o) {
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const int i = b0 + lane;
    const int rows = (i < p.B ? min(max(p.cu[i + 1] - p.cu[i], 0), p.max_q) : 0) * p.G;
    const int nb = rows > p.small ? (rows + R - 1) / R : 0;
    int sum = nb;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    const unsigned above = __ballot_sync(0xffffffffu, sum > bx);
    if (above) {
      const int src = __ffs(above) - 1;
      return paged_block_of<R>(p, b0 + src, (bx - __shfl_sync(0xffffffffu, sum - nb, src)) * R, lane, o);
    }
    bx -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

__device__ __forceinline__ int paged_parts(const PagedAttnParams& p, int kend) {
  return max(1, (kend + p.span - 1) / p.span);
}

// ---------------------------------------------------------------------------
// up to 16 rows: mma.sync
// ---------------------------------------------------------------------------
// A CTA of 4 warps takes 16 rows of one (sequence, KV head) over one part of
// the keys; warp w the 16-key tiles w, w + 4, ...  A tile lies in one page.  Its
// K and V rows come by 16-byte cp.async into buffers of the warp's own, 16 KB in
// flight a warp, so no barrier is needed inside the loop.  S = Q K^T and
// O += P V run on m16n8k16 with fp32 sums; P enters as a bf16 pair hi + lo.
//
// int8: codes become bf16 exactly in registers.  For the byte u of a code,
// bf16 128 + (u & 127) and 128 + (u & 128) are both bit patterns
// (0x4300 | bits), and their difference is the code: three instructions for two
// codes.  The order of dims (S) and of output columns (O) is permuted so that
// each thread's bytes are what its fragments need.  The keys' scales multiply
// the scores, the values' scales the probabilities.
constexpr int PRA_R = 16;
constexpr int PRA_TILE = 16;
constexpr int PRA_WARPS = 4;
constexpr int PRA_THREADS = PRA_WARPS * 32;

template <int D, bool I8>
struct PraShape {
  static constexpr int ROW = D * (I8 ? 1 : 2);           // bytes of a row
  static constexpr int CPR = ROW / 16;                   // 16-byte chunks of a row
  static constexpr int HALF = PRA_TILE * ROW;            // K (or V) of a tile
  static constexpr int BUF = 2 * HALF + (I8 ? 128 : 0);  // + 16 key and 16 value scales
  static constexpr int NBUF = 8192 / HALF;
  static constexpr int SMEM_TILES = PRA_WARPS * NBUF * BUF;
  static constexpr int SMEM_MERGE = PRA_WARPS * PRA_R * (D + 2) * 4;
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

__device__ __forceinline__ uint32_t bf2_sub(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// the codes in bytes 0 and 2 of w as a bf16 pair
__device__ __forceinline__ uint32_t codes_bf2(uint32_t w) {
  return bf2_sub((w & 0x007F007Fu) | 0x43004300u, (w & 0x00800080u) | 0x43004300u);
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

template <int D, bool I8>
__global__ void __launch_bounds__(PRA_THREADS, 3) paged_rows_kernel(const PagedAttnParams p) {
  using S = PraShape<D, I8>;
  extern __shared__ __align__(128) uint8_t smem_pra[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  pdl_wait();
  PagedBlock blk;
  if (!paged_block_direct<PRA_R>(p, blockIdx.x, lane, blk)) return;
  const int g = blockIdx.y, sp = blockIdx.z;
  const int nparts = paged_parts(p, blk.kend);
  if (sp >= nparts) return;
  const int k0 = sp * p.span, k1 = min(blk.kend, k0 + p.span);  // this part's keys
  const int ntiles = max(0, (k1 - k0 + PRA_TILE - 1) / PRA_TILE);
  const int ntw = ntiles > warp ? (ntiles - warp + PRA_WARPS - 1) / PRA_WARPS : 0;
  const uint32_t buf0 = smem_u32(smem_pra) + warp * S::NBUF * S::BUF;
  const int32_t* table = p.kv.table + (size_t)blk.b * p.kv.max_pages;
  const int slot_mask = (1 << p.kv.page_shift) - 1;

  int pages = -1;  // lane l: the page of this warp's tile (i / 32) * 32 + l
  auto issue = [&](int i) {
    if ((i & 31) == 0) {
      const int t0 = k0 + (warp + (i + lane) * PRA_WARPS) * PRA_TILE;
      pages = -1;
      if (t0 < k1) {
        pages = table[t0 >> p.kv.page_shift];
        if (pages < 0 || pages >= p.kv.num_pages) {
          record_error(DEV_ERR_BOUNDS, 351);
          pages = -1;
        }
      }
    }
    const int page = __shfl_sync(0xffffffffu, pages, i & 31);
    const int t0 = k0 + (warp + i * PRA_WARPS) * PRA_TILE;
    const int nk = page < 0 ? 0 : min(PRA_TILE, k1 - t0);
    const size_t row0 = paged_row(p.kv, max(page, 0), g, t0 & slot_mask);
    const uint32_t base = buf0 + (i % S::NBUF) * S::BUF;
#pragma unroll
    for (int k = 0; k < S::CPR; ++k) {
      const int x = lane + 32 * k;
      const bool is_v = x >= PRA_TILE * S::CPR;
      const int row = (x / S::CPR) % PRA_TILE, c = x % S::CPR;
      const uint8_t* src = (is_v ? p.kv.v : p.kv.k) + (row0 + (row < nk ? row : 0)) * S::ROW + c * 16;
      const uint32_t off = is_v ? S::HALF + pra_off<S::CPR, false>(row, c) : pra_off<S::CPR, I8>(row, c);
      cp_async16_zfill(base + off, src, row < nk ? 16u : 0u);
    }
    if (I8) {
      const int row = lane & 15;
      const float* src = (lane < 16 ? p.kv.ks : p.kv.vs) + row0 + (row < nk ? row : 0);
      cp_async4_zfill(base + 2 * S::HALF + lane * 4, src, row < nk ? 4u : 0u);
    }
  };
#pragma unroll
  for (int i = 0; i < S::NBUF; ++i) {
    if (i < ntw) issue(i);
    cp_async_commit();
  }

  // query fragments of rows qr and qr + 8
  const int qr = lane >> 2, qc = lane & 3;
  uint32_t qa[D / 16][4];
  int lim[2];  // keys that the two rows see
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = blk.row0 + qr + 8 * h;
    const bool in = qr + 8 * h < blk.nrows;
    const int tok = r / p.G, head = g * p.G + r - tok * p.G;
    lim[h] = in ? blk.past + tok + 1 : 0;
    const uint16_t* row = p.q + (size_t)(blk.tok0 + (in ? tok : 0)) * p.ld_q + (in ? head : 0) * D;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      if (I8) {
        // dims 64 (ks / 4) + 16 qc + 4 (ks % 4) + e: e = 0, 2 in the first pair, 1, 3 in the second
        uint2 w = make_uint2(0, 0);
        if (in) w = *reinterpret_cast<const uint2*>(row + 64 * (ks / 4) + 16 * qc + 4 * (ks % 4));
        qa[ks][h] = __byte_perm(w.x, w.y, 0x5410);
        qa[ks][2 + h] = __byte_perm(w.x, w.y, 0x7632);
      } else {
        qa[ks][h] = in ? *reinterpret_cast<const uint32_t*>(row + 16 * ks + 2 * qc) : 0u;
        qa[ks][2 + h] = in ? *reinterpret_cast<const uint32_t*>(row + 16 * ks + 8 + 2 * qc) : 0u;
      }
    }
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
  const int mi = lane >> 3, mr = lane & 7;

  for (int i = 0; i < ntw; ++i) {
    cp_async_wait<S::NBUF - 1>();
    __syncwarp();
    const uint32_t kb = buf0 + (i % S::NBUF) * S::BUF, vb = kb + S::HALF;
    const int t0 = k0 + (warp + i * PRA_WARPS) * PRA_TILE;
    float s[2][4];  // keys 8 n + 2 qc, + 1 of rows qr (0, 1) and qr + 8 (2, 3)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
    if (I8) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          uint32_t w[4];
          const uint32_t a = kb + pra_off<S::CPR, true>(8 * n + qr, 4 * h + qc);
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_bf16_16816_full(s[n], qa[4 * h + k][0], qa[4 * h + k][1], qa[4 * h + k][2], qa[4 * h + k][3],
                                codes_bf2(w[k]), codes_bf2(w[k] >> 8));
        }
    } else {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4(kb + pra_off<S::CPR, false>((mi >> 1) * 8 + mr, 2 * ks + (mi & 1)), b0, b1, b2, b3);
        mma_bf16_16816_full(s[0], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b0, b1);
        mma_bf16_16816_full(s[1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b2, b3);
      }
    }
    float2 kscale[2], vscale[2];
    if (I8) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint32_t a = kb + 2 * S::HALF + (8 * n + 2 * qc) * 4;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(kscale[n].x), "=f"(kscale[n].y) : "r"(a));
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(vscale[n].x), "=f"(vscale[n].y) : "r"(a + 64));
      }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = t0 + 8 * n + 2 * qc + (e & 1);
        float x = s[n][e] * p.scale_log2;
        if (I8) x *= (e & 1) ? kscale[n].y : kscale[n].x;
        s[n][e] = key < lim[e >> 1] ? x : -INFINITY;
        mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
      }
    float corr[2], ref[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
      const float mn = fmaxf(m[h], mx[h]);
      ref[h] = mn == -INFINITY ? 0.f : mn;  // a row that has seen no key yet
      corr[h] = exp2f(m[h] - ref[h]);
      m[h] = mn;
      l[h] *= corr[h];
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = s[n][e];
        float w = exp2f(x - ref[e >> 1]);
        l[e >> 1] += w;
        // a masked key's scale may be anything
        if (I8) w = x == -INFINITY ? 0.f : w * ((e & 1) ? vscale[n].y : vscale[n].x);
        s[n][e] = w;
      }
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      o[j][0] *= corr[0];
      o[j][1] *= corr[0];
      o[j][2] *= corr[1];
      o[j][3] *= corr[1];
    }
    uint32_t ph[4], pl[4];  // (row qr, keys 2 qc), (qr + 8, 2 qc), (qr, 8 + 2 qc), (qr + 8, 8 + 2 qc)
    split_bf2(s[0][0], s[0][1], ph[0], pl[0]);
    split_bf2(s[0][2], s[0][3], ph[1], pl[1]);
    split_bf2(s[1][0], s[1][1], ph[2], pl[2]);
    split_bf2(s[1][2], s[1][3], ph[3], pl[3]);
#pragma unroll
    for (int jj = 0; jj < S::CPR / 2; ++jj) {
      // transposed 8 x 8 matrices: (keys 0-7, chunk 2 jj), (keys 8-15, 2 jj), (keys 0-7, 2 jj + 1), (keys 8-15, 2 jj + 1)
      uint32_t b0, b1, b2, b3;
      ldsm_x4_t(vb + pra_off<S::CPR, false>((mi & 1) * 8 + mr, 2 * jj + (mi >> 1)), b0, b1, b2, b3);
      if (I8) {
        // a chunk holds 16 dims: its even dims are one n-tile, its odd dims the next
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t x0 = c ? b2 : b0, x1 = c ? b3 : b1;
#pragma unroll
          for (int odd = 0; odd < 2; ++odd) {
            const uint32_t v0 = codes_bf2(odd ? x0 >> 8 : x0), v1 = codes_bf2(odd ? x1 >> 8 : x1);
            float(&acc)[4] = o[4 * jj + 2 * c + odd];
            mma_bf16_16816_full(acc, ph[0], ph[1], ph[2], ph[3], v0, v1);
            mma_bf16_16816_full(acc, pl[0], pl[1], pl[2], pl[3], v0, v1);
          }
        }
      } else {
        mma_bf16_16816_full(o[2 * jj], ph[0], ph[1], ph[2], ph[3], b0, b1);
        mma_bf16_16816_full(o[2 * jj + 1], ph[0], ph[1], ph[2], ph[3], b2, b3);
        mma_bf16_16816_full(o[2 * jj], pl[0], pl[1], pl[2], pl[3], b0, b1);
        mma_bf16_16816_full(o[2 * jj + 1], pl[0], pl[1], pl[2], pl[3], b2, b3);
      }
    }
    __syncwarp();
    if (i + S::NBUF < ntw) issue(i + S::NBUF);
    cp_async_commit();
  }
  cp_async_wait<0>();
  __syncthreads();  // the tiles' memory is free

  // the warps' states: [warp][row] (m, l), then [warp][row][D]
  float2* sm_ml = reinterpret_cast<float2*>(smem_pra);
  float* sm_o = reinterpret_cast<float*>(sm_ml + PRA_WARPS * PRA_R);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (qc == 0) sm_ml[warp * PRA_R + qr + 8 * h] = make_float2(m[h], l[h]);
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      // int8: n-tile j holds the dims of parity j % 2 of chunk j / 2
      const int d = I8 ? 16 * (j >> 1) + 4 * qc + (j & 1) : 8 * j + 2 * qc;
      float* dst = sm_o + (size_t)(warp * PRA_R + qr + 8 * h) * D + d;
      dst[0] = o[j][2 * h];
      dst[I8 ? 2 : 1] = o[j][2 * h + 1];
    }
  }
  __syncthreads();
  const size_t pb = ((size_t)sp * p.blocks + blockIdx.x) * p.kv.n_kv + g;
  for (int idx = tid; idx < blk.nrows * (D / 4); idx += PRA_THREADS) {
    const int r = idx / (D / 4), d = (idx % (D / 4)) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < PRA_WARPS; ++w) M = fmaxf(M, sm_ml[w * PRA_R + r].x);
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
#pragma unroll
    for (int w = 0; w < PRA_WARPS; ++w) {
      const float2 ml = sm_ml[w * PRA_R + r];
      const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
      const float4 a = *reinterpret_cast<const float4*>(sm_o + (size_t)(w * PRA_R + r) * D + d);
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
      if (d == 0) p.part_ml[pb * PRA_R + r] = make_float2(M, den);
      *reinterpret_cast<float4*>(p.part_o + (pb * PRA_R + r) * D + d) = num;
    }
  }
}

// ---------------------------------------------------------------------------
// joining the parts
// ---------------------------------------------------------------------------
// One warp a row: weighs the parts' unnormalised outputs by exp2(m_part - max).
// A block whose keys fit in one part was written by its own CTA.
template <int D, int R>
__global__ void __launch_bounds__(128) paged_join_kernel(const PagedAttnParams p) {
  const int lane = threadIdx.x & 31, r = blockIdx.z * 4 + (threadIdx.x >> 5), g = blockIdx.y;
  pdl_trigger();
  pdl_wait();
  PagedBlock blk;
  if (!(R == PRA_R ? paged_block_direct<R>(p, blockIdx.x, lane, blk) : paged_block_search<R>(p, blockIdx.x, lane, blk)))
    return;
  const int nparts = paged_parts(p, blk.kend);
  if (nparts == 1 || r >= blk.nrows) return;
  const size_t step = (size_t)p.blocks * p.kv.n_kv;
  const size_t pb = (size_t)blockIdx.x * p.kv.n_kv + g;
  float M = -INFINITY;
  for (int s = lane; s < nparts; s += 32) M = fmaxf(M, p.part_ml[(pb + s * step) * R + r].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  constexpr int V = D / 32;
  float num[V], den = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) num[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < nparts; ++s) {
    const size_t at = (pb + s * step) * R + r;
    const float2 ml = p.part_ml[at];
    const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
    den = fmaf(ml.y, f, den);
#pragma unroll
    for (int e = 0; e < V; ++e) num[e] = fmaf(p.part_o[at * D + lane * V + e], f, num[e]);
  }
  const float inv = M == -INFINITY ? 0.f : 1.f / den;
  const int row = blk.row0 + r, tok = row / p.G;
  uint32_t* dst = reinterpret_cast<uint32_t*>(
      p.out + ((size_t)(blk.tok0 + tok) * p.n_heads + g * p.G + row - tok * p.G) * D + lane * V);
#pragma unroll
  for (int e = 0; e < V / 2; ++e) dst[e] = bf2_of(num[2 * e] * inv, num[2 * e + 1] * inv);
}

}  // namespace bitnet
