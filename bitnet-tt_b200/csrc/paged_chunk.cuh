// Attention of chunks of new tokens over paged keys and values, on the tcgen05
// tensor cores (what paged_attention.cuh says of rows, blocks and parts holds).
//
// A CTA takes up to 256 packed rows of one (sequence, KV head), as two tiles of
// 128 rows, over one part of the keys, 64 keys a step:
//   S_t = Q_t K^T     128 x 64 fp32 in tensor memory, Q_t and K from shared memory
//   P_t = exp2(scale log2(e) S_t - m), written over S_t as 16-bit floats
//   O_t += P_t V      P_t from tensor memory, V (keys x dims) from shared memory
// Tensor memory (512 columns) holds two S of each row tile and the two O.  So S of
// the next step is there when the softmax of one is done, and neither waits for
// the other: with one S of 128 keys a tile, the products that follow a softmax and
// the signals between them (about 1300 cycles) stood in every step's chain, and
// two 4096-token chunks over 16384 keys took 690 us (589 now, 1167 TFLOP/s; int8
// 824).  What bounds a step now (1670 cycles, int8 2150) is a tile's softmax chain
// beside the MMAs: 190 until it sees the scores, 230 to load them, 330 for the
// maximum, 790 for exponentials, sums and P; the MMAs alone take 1280 and the
// softmax of both tiles alone 1000.  The price of short steps is that 64-key
// score products read Q twice as often: 48 cycles each (shared memory's rate)
// instead of half of 64.
// Roles, one warp each unless said otherwise:
//   warps 0-3, 4-7   softmax of tile 0 and of tile 1: a thread owns a row (a lane of
//                    tensor memory), so maxima and sums need no shuffles
//   warps 8, 9       issue the MMAs of tile 0 and of tile 1: O_t of a step, then S_t of the step
//                    after next.  Two, because the tensor cores queue few MMAs: a look at a
//                    barrier costs the issuing warp about 100 cycles even when it is complete,
//                    and with one warp those were gaps (980 cycles a tile and step for 640 of work)
//   warp 10          loads K and V tiles by TMA, a box per page, into a ring of slots (int8: of
//                    raw tiles)
//   warps 12-15 (int8)  write the raw tiles' codes to the slots as f16
// The softmax's maximum is lazy: O and the sum are rescaled only when a row's
// maximum grew by more than 2^8, so weights reach at most 2^8 and the pass over
// O is rare (it waits for the products in flight); sums and outputs are fp32.  The
// exponentials are what a tile costs most: 16 a cycle and SM against 4096 products.
// A quarter of them is therefore computed on the multiply-add units (ex2_poly2).
//
// P of a sequence of more than 32 rows is one bf16 (half a step: 2^-8 of a weight), the
// output's own precision; the sums take the weights before they are rounded.  The two
// 4096-token chunks come out within 2.2e-3 of the exact result (norms).  With a pair
// hi + lo, 16 bits, for all they come within 1.65e-3, which is the output's rounding
// alone, but took 752 us where one bf16 took 570: the second product per step adds to
// the MMAs.  A third of the time for an error that stays below the output's own step
// is not taken.  Sequences of up to 32 rows (drafted tokens that stand beside chunks)
// get the pair and no polynomial: alone they go to paged_rows_kernel, which works to
// the same precision.  2 chunks of 1024 beside 30 x 5 tokens over 4096 keys: 170 us
// with it, 159 without.
//
// int8: everything is f16.  The keys' codes are f16 values exactly, and their
// scales multiply the scores in fp32, where an error would be raised to a power.
// The values are code * scale, the scale and the product rounded to f16 (2^-11 each) at
// a power of two taken from the largest scale of the part, which keeps rows down to
// 2^-21 of it at that precision, and smaller ones to 2^-32 of 127 times it.  Q is scaled
// by a power of two per row (exact), P has f16's 11 bits.
// Codes come out of their words as (0, 2) and (1, 3) pairs, so every four dims of
// the slots stand in the order 0, 2, 1, 3: Q is laid out the same way, and the
// output is put back when it is stored.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "paged_attention.cuh"

namespace bitnet {

constexpr int PCH_R = 256;   // rows of a CTA
constexpr int PCH_KB = 128;  // keys of a tile (a slot of K or V)
constexpr int PCH_STEP = 64; // keys of a step
constexpr int PCH_MAX_SLOTS = 8;
constexpr float PCH_GROWTH = 8.f;

template <int D, bool I8>
struct PchShape {
  static constexpr int THREADS = I8 ? 512 : 352;
  static constexpr int TILE = 128 * D * 2;          // bytes of Q_t, K or V as bf16
  static constexpr int NSLOT = D == 64 ? 8 : (I8 ? 4 : 5);
  // int8: the keys' scales [RING tiles][128], then the rows' factors [256].  When the codes of
  // key tile j are in their slot, the value slot of tile j - RING has been released, after both
  // softmaxes of that tile.
  static constexpr int RING = NSLOT / 2 + 1;
  static constexpr int EXTRA = I8 ? RING * 512 + 1024 : 0;
  // int8: raw tiles in flight.  (Loaded through the converting warps' registers, one tile ahead,
  // the loads' latency was what a step cost: 913 us where this takes 851, two 4096-token chunks over
  // 16384 keys.)
  static constexpr int NRAW = I8 ? (D == 64 ? 4 : 2) : 0, RAW = 128 * D;
  // Weights are exp2(x - m + LIFT): with f16's range the smallest step is below 2^-31 of the largest.
  static constexpr float LIFT = I8 ? 7.f : 0.f;
  // int8: registers a thread of the softmax, MMA and converting warpgroups, out of the launch's 128
  static constexpr int REGS_SOFTMAX = 176, REGS_MMA = 56, REGS_CONVERT = 104;
  static_assert(256 * REGS_SOFTMAX + 128 * REGS_MMA + 128 * REGS_CONVERT <= 512 * 128, "within the launch's");
  static constexpr int CTRL = 512;
  static constexpr int SMEM = 2 * TILE + NSLOT * TILE + NRAW * RAW + EXTRA + CTRL;
};

// One lane of a converged warp.  The MMAs and their commits are issued under it:
// under `lane == 0` the compiler has to allow for several lanes with different
// operands, and an MMA took about 75 cycles to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// 2^y for two values without the exponential unit: n = round(y) by adding 1.5 * 2^23,
// 2^(y - n) by a cubic (fitted for the least largest relative error on [-1/2, 1/2]:
// 7.5e-5, a fiftieth of a bf16's half step, a sixth of an f16's), times 2^n by its bits.
// y is held at -127 and above, where 2^n is 0: so is the weight of a hidden key, and a
// NaN stays one.  (n added to the cubic's exponent is an operation less a pair, but leaves
// a hidden key 2^-126, which a large value can raise to anything, and makes a NaN 3e38.)
__device__ __forceinline__ void ex2_poly2(uint64_t y, float& a, float& b) {
  uint32_t lo, hi;
  f2_split(y, lo, hi);
  float x0, x1;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x0) : "f"(__uint_as_float(lo)), "f"(-127.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x1) : "f"(__uint_as_float(hi)), "f"(-127.f));
  y = f2_make(__float_as_uint(x0), __float_as_uint(x1));
  const uint64_t t = f2_add(y, f2_splat(12582912.f));
  const uint64_t f = f2_fma(f2_add(t, f2_splat(-12582912.f)), f2_splat(-1.f), y);
  uint64_t p = f2_fma(f2_splat(0.05517166852951050f), f, f2_splat(0.2426111251115799f));
  p = f2_fma(p, f, f2_splat(0.6932609677314758f));
  p = f2_fma(p, f, f2_splat(0.9999280571937561f));
  uint32_t t0, t1;
  f2_split(t, t0, t1);
  uint32_t w0, w1;
  f2_split(f2_mul(p, f2_make((t0 << 23) + 0x3f800000u, (t1 << 23) + 0x3f800000u)), w0, w1);
  a = __uint_as_float(w0);
  b = __uint_as_float(w1);
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The exponent field of the power of two 2^k / 2^floor(log2 x), x by its fp32 bits.
__device__ __forceinline__ uint32_t pow2_field(uint32_t bits, int k) { return 254u + k - max(bits >> 23, 32u); }

struct PchCtrl {
  uint64_t full[PCH_MAX_SLOTS], empty[PCH_MAX_SLOTS];
  uint64_t raw_full[4], raw_empty[4];
  uint64_t s_full[2][2], p_ready[2][2];  // [row tile][step % 2]
  uint64_t o_done[2][2], drain[2], tail, q_full, v_full;  // o_done: O_t holds the step
  uint32_t tmem;
  int abort_flag;
  uint32_t v_top[4];  // int8: the largest value scale of the part, by its bits, as each converting warp saw it
  PagedBlock block;   // nrows 0: none
};
static_assert(sizeof(PchCtrl) <= 512, "control block");

template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
// 128-byte swizzled tile: rows of 128 bytes, 8 rows an atom of 1024 bytes.
//   K major (Q, K): sbo = the next 8 rows; lbo unused
//   MN major (V):   lbo = the next 64 dims, sbo = the next 8 keys
__device__ __forceinline__ uint64_t smem_desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)((lbo >> 4) & 0x3FFFu) << 16 |
         (uint64_t)((sbo >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D[tmem] (+)= A[tmem] x B[smem], bf16 x bf16 -> fp32
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 32 lanes x 32 columns of 32 bits
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ uint32_t pch_v_top(const PchCtrl* c) {
  uint32_t t = c->v_top[0];
  for (int i = 1; i < 4; ++i) t = max(t, c->v_top[i]);
  return t;
}

template <int D, bool I8>
__global__ void __launch_bounds__(PchShape<D, I8>::THREADS, 1)
    paged_chunk_kernel(const PagedAttnParams p, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v) {
  using S = PchShape<D, I8>;
  constexpr int HALF = 128 * 128;  // bytes of 64 dims of a tile
  extern __shared__ __align__(1024) uint8_t smem_pch[];
  uint8_t* sm_q = smem_pch;
  uint8_t* sm_slots = sm_q + 2 * S::TILE;
  uint8_t* sm_raw = sm_slots + S::NSLOT * S::TILE;
  float* sm_scale = reinterpret_cast<float*>(sm_raw + S::NRAW * S::RAW);
  float* sm_fac = sm_scale + S::RING * 128;
  PchCtrl* ctrl = reinterpret_cast<PchCtrl*>(sm_raw + S::NRAW * S::RAW + S::EXTRA);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &ctrl->abort_flag;
  if (tid == 0) {
    for (int s = 0; s < S::NSLOT; ++s) {
      mbar_init(&ctrl->full[s], I8 ? 4 : 1);
      mbar_init(&ctrl->empty[s], 2);
    }
    for (int s = 0; s < S::NRAW; ++s) {
      mbar_init(&ctrl->raw_full[s], 1);
      mbar_init(&ctrl->raw_empty[s], 4);
    }
    for (int t = 0; t < 2; ++t) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&ctrl->s_full[t][h], 1);
        mbar_init(&ctrl->p_ready[t][h], 4);
        mbar_init(&ctrl->o_done[t][h], 1);
      }
      mbar_init(&ctrl->drain[t], 1);
    }
    mbar_init(&ctrl->tail, 1);
    mbar_init(&ctrl->q_full, 8);
    mbar_init(&ctrl->v_full, 4);
    ctrl->abort_flag = 0;
    fence_mbar_init();
  }
  pdl_wait();
  // The rows kernel may then start without a wait of its own.  What the wait made visible is published first,
  // once: a fence in every CTA delays those that have no block (16 chunks beside 240 int8 rows: 195 -> 204 us).
  if (blockIdx.x > 0) {
    pdl_trigger();
  } else if (tid == 0) {
    fence_acq_rel_gpu();
    pdl_trigger();
  }
  // Blocks vary slowest: CTAs start in this order, and the longest blocks of all heads come first.
  const int g = blockIdx.x % p.kv.n_kv, bs = blockIdx.x / p.kv.n_kv, bx = bs / p.nsplit, sp = bs - bx * p.nsplit;
  // One warp searches: the code is cold, and all warps at it took longer than one and the exchange.
  // Tensor memory after pdl_wait: the kernel before this one may need it to end.  (A later kernel cannot
  // hold it, waiting for this one: the kernels that do need 15,000 registers or more, and beside a CTA of
  // this one an SM has 6,400.)
  if (warp == 8) {
    PagedBlock found;
    if (!paged_block_search<PCH_R>(p, bx, lane, found)) found.nrows = 0;
    if (lane == 0) {
      ctrl->block = found;
      if (p.nsplit > 1 && sp == 0 && g == 0) p.found[bx] = found;  // for the join
    }
    __syncwarp();  // lane 0 was apart: tensor memory is taken, read and written by whole warps
    if (found.nrows > 0 && sp < paged_parts(p, found.kend)) {
      tmem_alloc(&ctrl->tmem, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const PagedBlock blk = ctrl->block;
  if (blk.nrows == 0) return;
  const int nparts = paged_parts(p, blk.kend);
  if (sp >= nparts) return;
  const int k0 = sp * p.span, k1 = min(blk.kend, k0 + p.span);
  const bool fine = !I8 && blk.row0 == 0 && blk.nrows <= PAGED_FINE;  // the whole sequence: weights as hi + lo
  // 64-key steps of the two row tiles (the second sees at least the first's keys)
  const int end0 = min(k1, max(0, blk.past + (blk.row0 + min(blk.nrows, 128) - 1) / p.G + 1));
  const int n0 = max(0, (end0 - k0 + PCH_STEP - 1) / PCH_STEP);
  const int n1 = blk.nrows > 128 ? max(0, (k1 - k0 + PCH_STEP - 1) / PCH_STEP) : 0;
  const int nstep = max(n0, n1), ntile = (nstep + 1) / 2;
  // All 512 columns are this CTA's, so they start at 0: a constant, as the MMAs' operands
  // should be (below).
  constexpr uint32_t tbase = 0;

  auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (!mbar_wait(bar, parity, site)) {
      *abort_flag = 1;
      return false;
    }
    return true;
  };

  if (I8 && warp >= 12) {
    // ---------------- int8: codes to f16 slots ----------------
    if constexpr (I8) {
      regs_dec<S::REGS_CONVERT>();
      constexpr int NL = D / 16;  // 16-byte loads of a lane: 32 rows of a warp
      const int w = warp - 12;
      const int32_t* table = p.kv.table + (size_t)blk.b * p.kv.max_pages;
      const int slot_mask = (1 << p.kv.page_shift) - 1;
      // this lane's row of a tile: the page, then the scales (0 past the part's keys)
      auto key_of = [&](int j) { return k0 + j * PCH_KB + 32 * w + lane; };
      auto page_of = [&](int j) {
        if (j >= ntile || key_of(j) >= k1) return -1;
        const int page = table[key_of(j) >> p.kv.page_shift];
        return page < p.kv.num_pages ? page : -1;  // a bad one is reported by the loader
      };
      auto scales_of = [&](int j, int page, float& ks, float& vs) {
        ks = vs = 0.f;
        if (page >= 0) {
          const size_t row = paged_row(p.kv, page, g, key_of(j) & slot_mask);
          ks = p.kv.ks[row];
          vs = p.kv.vs[row];
        }
      };
      // Raw tile `it` to its slot; scale: of this lane's row of the warp's 32, as f16 (values only).
      // Row and 16-byte chunk of piece u are such that eight lanes read 128 bytes of different
      // banks and write eight different chunks.
      auto convert = [&](int it, uint32_t scale) -> bool {
        const int slot = it % S::NSLOT, stage = it % S::NRAW;
        bool ok = wait(&ctrl->raw_full[stage], (it / S::NRAW) & 1, 378);
        if (!__all_sync(0xffffffffu, ok)) return false;
        uint4 buf[NL];
        auto place = [&](int u, int& row, int& c) {
          if (D == 128) {
            c = lane & 7;
            row = 2 * ((u >> 1) * 4 + (lane >> 3)) + (((lane >> 2) & 1) ^ (u & 1));
          } else {
            c = lane & 3;
            row = u * 8 + (lane >> 2);
          }
        };
#pragma unroll
        for (int u = 0; u < NL; ++u) {
          int row, c;
          place(u, row, c);
          buf[u] = *reinterpret_cast<const uint4*>(sm_raw + stage * S::RAW + (32 * w + row) * D + c * 16);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctrl->raw_empty[stage]);
        if (it >= S::NSLOT && !__all_sync(0xffffffffu, wait(&ctrl->empty[slot], ((it / S::NSLOT) + 1) & 1, 362)))
          return false;
        uint8_t* dst = sm_slots + slot * S::TILE;
        const bool scaled = it & 1;
#pragma unroll
        for (int u = 0; u < NL; ++u) {
          int row, c;
          place(u, row, c);
          const uint32_t sc = scaled ? __shfl_sync(0xffffffffu, scale, row) : 0u;
          row += 32 * w;
          uint8_t* at = dst + (c >> 2) * HALF + row * 128;
          const uint32_t x[4] = {buf[u].x, buf[u].y, buf[u].z, buf[u].w};
          uint32_t y[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[2 * e] = codes_f2(x[e]), y[2 * e + 1] = codes_f2(x[e] >> 8);
          if (scaled) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = h2_mul(y[e], sc);
          }
          *reinterpret_cast<uint4*>(at + (((2 * (c & 3)) ^ (row & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
          *reinterpret_cast<uint4*>(at + (((2 * (c & 3) + 1) ^ (row & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
        }
        return true;
      };
      auto arrive = [&](int it) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctrl->full[it % S::NSLOT]);
      };
      float v_up = 0.f, ks, vs;
      scales_of(0, page_of(0), ks, vs);
      int page = page_of(1);
      for (int j = 0; j < ntile; ++j) {
        float ks1, vs1;
        scales_of(j + 1, page, ks1, vs1);  // the next tile's, on the way while this one is converted
        page = page_of(j + 2);
        if (!convert(2 * j, 0)) break;
        sm_scale[(j % S::RING) * 128 + 32 * w + lane] = ks;
        arrive(2 * j);
        if (j == 0) {  // the largest value scale of the part's rows, four rows (of one page) a load
          float top = 0.f;
#pragma unroll 4
          for (int key = k0 + 4 * (32 * w + lane); key < k1; key += 512) {
            const int at = table[key >> p.kv.page_shift];
            if (at < 0 || at >= p.kv.num_pages) continue;  // reported by the loader
            const float4 v = *reinterpret_cast<const float4*>(p.kv.vs + paged_row(p.kv, at, g, key & slot_mask));
            top = fmaxf(top, v.x);
            if (key + 1 < k1) top = fmaxf(top, v.y);
            if (key + 2 < k1) top = fmaxf(top, v.z);
            if (key + 3 < k1) top = fmaxf(top, v.w);
          }
          const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
          if (lane == 0) {
            ctrl->v_top[w] = most;
            mbar_arrive(&ctrl->v_full);
          }
          if (!__all_sync(0xffffffffu, wait(&ctrl->v_full, 0, 376))) break;
          v_up = __uint_as_float(pow2_field(pch_v_top(ctrl), 7) << 23);
        }
        if (!convert(2 * j + 1, f16x2_of(vs * v_up, vs * v_up))) break;
        arrive(2 * j + 1);
        ks = ks1, vs = vs1;
      }
    }
  } else if (warp >= 8) {
    if constexpr (I8) regs_dec<S::REGS_MMA>();
    const int t = warp == 8 ? 0 : 1, nt = t ? n1 : n0;
    if (warp < 10 && nstep > 0) {
      // ---------------- MMA issuers ----------------
      constexpr uint32_t f16_types = (1u << 7) | (1u << 10);  // set: bf16, clear: f16
      constexpr uint32_t idesc_s = idesc_bf16_f32(128, PCH_STEP) & (I8 ? ~f16_types : ~0u);
      constexpr uint32_t idesc_o = (idesc_bf16_f32(128, D) & (I8 ? ~f16_types : ~0u)) | (1u << 16);  // V: dims contiguous
      // descriptors of the first product: the others differ in the address field (16-byte units)
      const uint64_t dq = smem_desc_sw128(smem_u32(sm_q) + t * S::TILE, 16, 1024),
                     dk = smem_desc_sw128(smem_u32(sm_slots), 16, 1024), dv = smem_desc_sw128(smem_u32(sm_slots), HALF, 1024);
      auto qk = [&](int slot, int h) {
        const uint64_t b = dk + slot * (S::TILE >> 4) + h * (PCH_STEP * 128 >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k >> 2) * HALF + (k & 3) * 32) >> 4;
          mma_f16_ss(tbase + t * 128 + h * 64, dq + off, b + off, idesc_s, k > 0);
        }
        tc_commit(&ctrl->s_full[t][h]);
      };
      auto pv = [&](int slot, int h, bool first, auto fine_tag) {
        const uint64_t b = dv + slot * (S::TILE >> 4) + h * (PCH_STEP * 128 >> 4);
        const uint32_t a = tbase + t * 128 + h * 64, d = tbase + 256 + t * D;
#pragma unroll
        for (int k = 0; k < PCH_STEP / 16; ++k) mma_f16_ts(d, a + k * 8, b + k * (16 * 128 >> 4), idesc_o, k > 0 || !first);
        if constexpr (decltype(fine_tag)::value) {
#pragma unroll
          for (int k = 0; k < PCH_STEP / 16; ++k) mma_f16_ts(d, a + 32 + k * 8, b + k * (16 * 128 >> 4), idesc_o, 1);
        }
        tc_commit(&ctrl->o_done[t][h]);
      };
      auto arrived = [&](uint64_t* bar, uint32_t parity, int site) {
        const bool ok = __all_sync(0xffffffffu, wait(bar, parity, site));
        tc_fence_after();
        return ok;
      };
      auto filled = [&](int it, int site) { return arrived(&ctrl->full[it % S::NSLOT], (it / S::NSLOT) & 1, site); };
      // Each issuer releases every slot, those past its own tile's keys too.
      bool ok = filled(0, 363) && arrived(&ctrl->q_full, 0, 375);
      if (ok && elect_one()) {
        if (nt > 0) qk(0, 0);
        if (nt > 1) qk(0, 1);
        tc_commit(&ctrl->empty[0]);
      }
      __syncwarp();
      auto steps = [&](auto fine_tag) {
        for (int i = 0; ok && i < nstep; ++i) {
          const int j = i >> 1, h = i & 1;
          const int vs = (2 * j + 1) % S::NSLOT, ks = (2 * j + 2) % S::NSLOT;  // slots of V, and of the next K
          if (h == 0) {
            ok = filled(2 * j + 1, 364);
            if (ok && i + 2 < nstep) ok = filled(2 * j + 2, 366);
          }
          if (ok && i < nt) ok = arrived(&ctrl->p_ready[t][h], j & 1, 365);
          if (ok && elect_one()) {
            if (i < nt) pv(vs, h, i == 0, fine_tag);
            if (i + 2 < nt) qk(ks, h);
            if (h == 1 || i + 1 == nstep) tc_commit(&ctrl->empty[vs]);
            if (i + 2 < nstep && (h == 1 || i + 3 == nstep)) tc_commit(&ctrl->empty[ks]);
          }
          __syncwarp();
        }
      };
      // two copies of the loop, as of the softmax's: a choice inside it costs the common one 16%
      if (fine) steps(std::true_type{});
      else steps(std::false_type{});
      if (!ok) {  // let the MMAs in flight end before tensor memory is freed
        if (elect_one()) tc_commit(&ctrl->drain[t]);
        __syncwarp();
        mbar_wait(&ctrl->drain[t], 0, 367);
      }
    } else if (warp == 10) {
      // ---------------- TMA loads ----------------
      const int32_t* table = p.kv.table + (size_t)blk.b * p.kv.max_pages;
      const int box = min(1 << p.kv.page_shift, PCH_KB);  // rows of a box: the map's
      const int slot_mask = (1 << p.kv.page_shift) - 1;
      int issued = 0;
      bool ok = true, tail_issued = false;
      for (int j = 0; ok && j < ntile; ++j) {
        const int base = k0 + j * PCH_KB;
        const int nbox = (min(k1 - base, PCH_KB) + box - 1) / box;  // boxes that hold keys
        int y = 0;
        if (lane < nbox) {
          const int key = base + lane * box;
          int page = table[key >> p.kv.page_shift];
          if (page < 0 || page >= p.kv.num_pages) {
            record_error(DEV_ERR_BOUNDS, 360);
            page = 0;
          }
          y = (int)paged_row(p.kv, page, g, key & slot_mask);
        }
        for (int v = 0; ok && v < 2; ++v) {
          const int it = 2 * j + v;
          if constexpr (I8) {
            // rows past the last key hold any codes: finite, and their scales are taken as 0
            const int stage = it % S::NRAW;
            if (it >= S::NRAW) ok = __all_sync(0xffffffffu, wait(&ctrl->raw_empty[stage], ((it / S::NRAW) + 1) & 1, 379));
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&ctrl->raw_full[stage], (uint32_t)(nbox * box * D));
            __syncwarp();
            if (lane < nbox)
              tma_load_2d(smem_u32(sm_raw + stage * S::RAW) + lane * box * D, v ? &map_v : &map_k, 0, y, &ctrl->raw_full[stage]);
            issued = it + 1;
          } else {
            const int slot = it % S::NSLOT;
            if (it >= S::NSLOT) ok = __all_sync(0xffffffffu, wait(&ctrl->empty[slot], ((it / S::NSLOT) + 1) & 1, 368));
            if (!ok) break;
            const bool tail = v == 1 && base + PCH_KB > k1;
            uint64_t* bar = tail ? &ctrl->tail : &ctrl->full[slot];
            if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(nbox * box * D * 2));
            __syncwarp();
            const uint32_t dst = smem_u32(sm_slots + slot * S::TILE) + lane * box * 128;
            if (lane < nbox) {
#pragma unroll
              for (int h = 0; h < D / 64; ++h) tma_load_2d(dst + h * HALF, v ? &map_v : &map_k, h * 64, y, bar);
            }
            issued = it + 1;
            if (tail) {
              tail_issued = true;
              // Whatever stands behind the last key must not meet a weight of 0: zeros.
              ok = __all_sync(0xffffffffu, wait(&ctrl->tail, 0, 369));
              if (!ok) break;
              const int live = k1 - base;
              for (int i = lane; i < (128 - live) * (D / 8); i += 32) {
                const int row = live + i / (D / 8), c = i % (D / 8);
                *reinterpret_cast<uint4*>(sm_slots + slot * S::TILE + (c >> 3) * HALF + row * 128 + ((c & 7) << 4)) =
                    make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&ctrl->full[slot]);
            }
          }
        }
      }
      if (*abort_flag) {  // copies in flight land before the CTA gives its memory back
        if constexpr (I8) {
          for (int it = max(0, issued - S::NRAW); it < issued; ++it)
            mbar_wait(&ctrl->raw_full[it % S::NRAW], (it / S::NRAW) & 1, 380);
        } else {
          if (tail_issued) mbar_wait(&ctrl->tail, 0, 370);
          for (int it = max(0, issued - S::NSLOT); it < issued - (tail_issued ? 1 : 0); ++it)
            mbar_wait(&ctrl->full[it % S::NSLOT], (it / S::NSLOT) & 1, 370);
        }
      }
    }
  } else {
    // ---------------- softmax: a thread owns a row (and the eight warps load Q first) ----------------
    if constexpr (I8) regs_inc<S::REGS_SOFTMAX>();
    // Q into the swizzled tiles by 16-byte asynchronous copies (rows past the block: zeros).  The
    // loops stay rolled: code that runs once a CTA comes from a cold instruction cache, and eight
    // unrolled loads took 6500 cycles (16500 with the conversion below).
    constexpr int RQ = 256 / (D / 8);  // rows between a thread's copies
    const int qc = tid % (D / 8), nq = blk.nrows > 128 ? 256 : 128;
    {
      int tok = (blk.row0 + tid / (D / 8)) / p.G, head = blk.row0 + tid / (D / 8) - tok * p.G;
      const int dt = RQ / p.G, dh = RQ - dt * p.G;
#pragma unroll 2
      for (int r = tid / (D / 8); r < nq; r += RQ) {
        const uint16_t* src = p.q + (size_t)(blk.tok0 + tok) * p.ld_q + (size_t)(g * p.G + head) * D + qc * 8;
        const bool in = r < blk.nrows;
        cp_async16_zfill(smem_u32(sm_q) + (r >> 7) * S::TILE + (qc >> 3) * HALF + (r & 127) * 128 + (((qc & 7) ^ (r & 7)) << 4),
                         in ? src : p.q, in ? 16u : 0u);
        tok += dt;
        head += dh;
        if (head >= p.G) head -= p.G, ++tok;
      }
    }
    cp_async_commit();
    cp_async_wait<0>();
    if (I8) {  // each thread its own chunks; D / 8 neighbouring lanes hold a row: its largest value goes to 2^13 .. 2^14
#pragma unroll 4
      for (int r = tid / (D / 8); r < nq; r += RQ) {
        uint4* at = reinterpret_cast<uint4*>(sm_q + (r >> 7) * S::TILE + (qc >> 3) * HALF + (r & 127) * 128 + (((qc & 7) ^ (r & 7)) << 4));
        float x[8];
        unpack_bf8(*at, x);
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
        for (int o = D / 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t field = pow2_field(top, 13);
        const float f = __uint_as_float(field << 23);
        *at = make_uint4(f16x2_of(x[0] * f, x[2] * f), f16x2_of(x[1] * f, x[3] * f), f16x2_of(x[4] * f, x[6] * f),
                         f16x2_of(x[5] * f, x[7] * f));
        if (qc == 0) sm_fac[r] = __uint_as_float((254u - field) << 23);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctrl->q_full);
    if (I8) {
      // sm_fac is read across warps
      named_bar_sync(1, 256);
    }
    const int t = warp >> 2, r = t * 128 + (warp & 3) * 32 + lane;
    const int nt = t ? n1 : n0;
    const bool live = r < blk.nrows;
    const bool warp_live = r - lane < blk.nrows;
    const int row = blk.row0 + r, tok = row / p.G;
    const int lim = live ? blk.past + tok + 1 : INT_MAX;
    const int lim_min = __reduce_min_sync(0xffffffffu, lim);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t to = tbase + lanes + 256 + t * D;
    // not 0, which a hidden key's -infinity must not meet
    const float scale = fmaxf(I8 ? p.scale_log2 * sm_fac[r] : p.scale_log2, 1e-37f);
    const uint64_t scale2 = f2_splat(scale);
    float m = -INFINITY;
    uint64_t l2[2] = {0, 0};
    bool ok = true;
    auto steps = [&](auto fine_tag) {
      constexpr bool FINE = decltype(fine_tag)::value;
      for (int i = 0; i < nt; ++i) {
        const int j = i >> 1, h = i & 1;
        ok = wait(&ctrl->s_full[t][h], j & 1, 371);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (warp_live) {
          const uint32_t ts = tbase + lanes + t * 128 + h * 64;
          uint32_t s[PCH_STEP];
          tmem_ld32(ts, s);
          tmem_ld32(ts + 32, s + 32);
          tmem_wait_ld();
          if (I8) {
            const ulonglong2* sc = reinterpret_cast<const ulonglong2*>(sm_scale + (j % S::RING) * 128 + h * 64);
#pragma unroll
            for (int c = 0; c < PCH_STEP / 4; ++c) {
              const ulonglong2 k = sc[c];
              f2_split(f2_mul(f2_make(s[4 * c], s[4 * c + 1]), k.x), s[4 * c], s[4 * c + 1]);
              f2_split(f2_mul(f2_make(s[4 * c + 2], s[4 * c + 3]), k.y), s[4 * c + 2], s[4 * c + 3]);
            }
          }
          const int base = k0 + i * PCH_STEP;
          if (base + PCH_STEP > min(lim_min, k1)) {
            const int see = min(lim, k1) - base;
#pragma unroll
            for (int c = 0; c < PCH_STEP; ++c)
              if (c >= see) s[c] = 0xff800000u;
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < PCH_STEP; c += 2)
            mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
          const float top = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * scale;
          if (i == 0) {
            m = top;
          } else if (__any_sync(0xffffffffu, top > m + PCH_GROWTH)) {
            const float mn = fmaxf(m, top);
            const float f = mn == -INFINITY ? 1.f : ex2(m - mn);
            m = mn;
            const uint64_t f2 = f2_splat(f);
            l2[0] = f2_mul(l2[0], f2);
            l2[1] = f2_mul(l2[1], f2);
            // O holds all steps so far once the product of step i - 1 is in (that of step i - 3, one
            // phase earlier on this barrier, is: S of step i - 1 came after it)
            ok = wait(&ctrl->o_done[t][h ^ 1], ((i - 1) >> 1) & 1, 374);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld32(to + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(to + c, o);
            }
          }
          const uint64_t ref2 = f2_splat(m == -INFINITY ? 0.f : S::LIFT - m);
#pragma unroll
          for (int c = 0; c < PCH_STEP; c += 32) {
            uint32_t pw[16], pl[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const uint64_t z = f2_fma(f2_make(s[c + 2 * e], s[c + 2 * e + 1]), scale2, ref2);
              float x, y;
              if (e % 4 == 3 && !FINE) {
                ex2_poly2(z, x, y);
              } else {
                uint32_t a, b;
                f2_split(z, a, b);
                x = ex2(__uint_as_float(a)), y = ex2(__uint_as_float(b));
              }
              l2[e & 1] = f2_add(l2[e & 1], f2_make(__float_as_uint(x), __float_as_uint(y)));
              if (FINE) split_bf2(x, y, pw[e], pl[e]);
              else pw[e] = I8 ? f16x2_of(x, y) : bf2_of(x, y);
            }
            tmem_st16(ts + c / 2, pw);
            if (FINE) tmem_st16(ts + 32 + c / 2, pl);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctrl->p_ready[t][h]);
      }
    };
    if (fine) steps(std::true_type{});
    else steps(std::false_type{});
    if (ok && nt > 0) ok = __all_sync(0xffffffffu, wait(&ctrl->o_done[t][(nt - 1) & 1], ((nt - 1) >> 1) & 1, 372));
    if (ok && warp_live) {
      tc_fence_after();
      uint32_t a, b, c2, d2;
      f2_split(l2[0], a, b);
      f2_split(l2[1], c2, d2);
      const float l = (__uint_as_float(a) + __uint_as_float(b)) + (__uint_as_float(c2) + __uint_as_float(d2));
      const bool sees = lim > 0;  // else zeros; by the mask, not by m, which is -infinity over NaN scores too
      const float inv = sees ? 1.f / l : 0.f;
      const size_t pr = (((size_t)sp * p.blocks + bx) * p.kv.n_kv + g) * PCH_R + r;
      if (live && nparts > 1) p.part_ml[pr] = make_float2(m - S::LIFT, l);
      if (I8 && nt > 0) wait(&ctrl->v_full, 0, 377);  // complete: the values were converted after it
      const float vf = I8 && nt > 0 ? __uint_as_float((254u - pow2_field(pch_v_top(ctrl), 7)) << 23) : 1.f;  // the values' power of two
      uint16_t* dst = p.out + ((size_t)(blk.tok0 + tok) * p.n_heads + g * p.G + row - tok * p.G) * D;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        __syncwarp();
        if (nt > 0) {
          tmem_ld32(to + c, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (I8) {  // the slots' dims back in order
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const uint32_t x = o[e + 1];
            o[e + 1] = o[e + 2];
            o[e + 2] = x;
          }
        }
        if (!live) continue;
        if (I8) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * vf);
        }
        if (nparts > 1) {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(p.part_o + pr * D + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = !sees ? 0u
                           : bf2_of(__uint_as_float(o[e + 2 * k]) * inv, __uint_as_float(o[e + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

}  // namespace bitnet
