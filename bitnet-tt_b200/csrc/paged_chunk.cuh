// Attention of chunks of new tokens over paged keys and values, on the tcgen05
// tensor cores (what paged_attention.cuh says of rows, blocks and parts holds).
//
// A CTA takes up to 256 packed rows of one (sequence, KV head), as two tiles of
// 128 rows, over one part of the keys, 128 keys at a time:
//   S_t = Q_t K^T     128 x 128 fp32 in tensor memory, Q_t and K from shared memory
//   P_t = exp2(scale log2(e) S_t - m), written over S_t as bf16
//   O_t += P_t V      P_t from tensor memory, V (keys x dims) from shared memory
// Roles, one warp each unless said otherwise:
//   warps 0-3, 4-7   softmax of tile 0 and of tile 1: a thread owns a row (a lane of
//                    tensor memory), so maxima and sums need no shuffles
//   warp 8           issues the MMAs: O_0, S_0 of the next keys, O_1, S_1; while one tile's
//                    products run, the other tile's softmax does
//   warp 9 (bf16)    loads K and V tiles by TMA, a box per page, into a ring of slots
//   warps 12-15 (int8)  load codes and write them to the slots as bf16 (exact)
// The softmax's maximum is lazy: O and the sum are rescaled only when a row's
// maximum grew by more than 2^8, so weights reach at most 2^8 and the pass over
// O is rare.  P is rounded to bf16 (half a step, 2^-9 of a weight on average
// less), the output's own precision; sums and outputs are fp32.
//
// int8: a code is a bf16 value, so the products see the codes exactly; the
// keys' scales multiply the scores, the values' scales the weights, both in
// fp32.  Codes come out of their words as (0, 2) and (1, 3) pairs, so every four
// dims of the slots stand in the order 0, 2, 1, 3: Q is laid out the same way,
// and the output is put back when it is stored.
#pragma once
#include <cuda.h>

#include "paged_attention.cuh"

namespace bitnet {

constexpr int PCH_R = 256;   // rows of a CTA
constexpr int PCH_KB = 128;  // keys of a tile
constexpr int PCH_MAX_SLOTS = 8;

template <int D, bool I8>
struct PchShape {
  static constexpr int THREADS = I8 ? 512 : 384;
  static constexpr int TILE = 128 * D * 2;          // bytes of Q_t, K or V as bf16
  static constexpr int NSLOT = D == 64 ? 8 : (I8 ? 4 : 5);
  // Scales [RING tiles][128 keys', 128 values'].  When the codes of key tile j are in their
  // slot, the value slot of tile j - RING has been released, after both softmaxes of that tile.
  static constexpr int RING = NSLOT / 2 + 1;
  static constexpr int SCALES = I8 ? RING * 1024 : 0;
  static constexpr int CTRL = 256;
  static constexpr int SMEM = 2 * TILE + NSLOT * TILE + SCALES + CTRL;
  // registers a thread: the launch gives 168 (384 threads) or 128 (512 threads)
  static constexpr int REGS_SOFTMAX = I8 ? 176 : 208;
  static constexpr int REGS_MMA = I8 ? 56 : 88;
  static constexpr int REGS_CONVERT = 104;
  static constexpr int REGS_LAUNCH = I8 ? 128 : 168;
};
static_assert(256 * 208 + 128 * 88 <= 384 * 168, "register shares within the launch's");
static_assert(256 * 176 + 128 * 56 + 128 * 104 <= 512 * 128, "register shares within the launch's");

__device__ __forceinline__ uint32_t bf2_sub(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// The codes in bytes 0 and 2 of w as a bf16 pair: for the byte u of a code,
// bf16 128 + (u & 127) and 128 + (u & 128) are both bit patterns (0x4300 | bits),
// and their difference is the code.
__device__ __forceinline__ uint32_t codes_bf2(uint32_t w) {
  return bf2_sub((w & 0x007F007Fu) | 0x43004300u, (w & 0x00800080u) | 0x43004300u);
}

struct PchCtrl {
  uint64_t full[PCH_MAX_SLOTS], empty[PCH_MAX_SLOTS];
  uint64_t s_full[2], p_ready[2], o_full[2], tail, drain;
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(PchCtrl) <= 256, "control block");

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
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
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
  float* sm_scale = reinterpret_cast<float*>(sm_slots + S::NSLOT * S::TILE);
  PchCtrl* ctrl = reinterpret_cast<PchCtrl*>(sm_slots + S::NSLOT * S::TILE + S::SCALES);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  pdl_wait();
  // the blocks with the most keys first
  PagedBlock blk;
  const int bx = p.blocks - 1 - (int)blockIdx.x;
  if (!paged_block_search<PCH_R>(p, bx, lane, blk)) return;
  const int g = blockIdx.y, sp = blockIdx.z;
  const int nparts = paged_parts(p, blk.kend);
  if (sp >= nparts) return;
  const int k0 = sp * p.span, k1 = min(blk.kend, k0 + p.span);
  // 128-key tiles of the two row tiles (the second sees at least the first's keys)
  const int end0 = min(k1, max(0, blk.past + (blk.row0 + min(blk.nrows, 128) - 1) / p.G + 1));
  const int n0 = max(0, (end0 - k0 + PCH_KB - 1) / PCH_KB);
  const int n1 = blk.nrows > 128 ? max(0, (k1 - k0 + PCH_KB - 1) / PCH_KB) : 0;
  const int ntile = max(n0, n1);

  volatile int* abort_flag = &ctrl->abort_flag;
  if (tid == 0) {
    for (int s = 0; s < S::NSLOT; ++s) {
      mbar_init(&ctrl->full[s], I8 ? 4 : 1);
      mbar_init(&ctrl->empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&ctrl->s_full[t], 1);
      mbar_init(&ctrl->p_ready[t], 4);
      mbar_init(&ctrl->o_full[t], 1);
    }
    mbar_init(&ctrl->tail, 1);
    mbar_init(&ctrl->drain, 1);
    ctrl->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(&ctrl->tmem, 512);
    tmem_relinquish();
  }
  // Q, 16 bytes at a time, into the swizzled tiles (rows past the block: zeros)
  for (int i = tid; i < 2 * 128 * (D / 8); i += S::THREADS) {
    const int r = i / (D / 8), c = i % (D / 8);
    if (r >= 128 && blk.nrows <= 128) break;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (r < blk.nrows) {
      const int row = blk.row0 + r, tok = row / p.G;
      w = *reinterpret_cast<const uint4*>(p.q + (size_t)(blk.tok0 + tok) * p.ld_q +
                                          (size_t)(g * p.G + row - tok * p.G) * D + c * 8);
      if (I8)
        w = make_uint4(__byte_perm(w.x, w.y, 0x5410), __byte_perm(w.x, w.y, 0x7632), __byte_perm(w.z, w.w, 0x5410),
                       __byte_perm(w.z, w.w, 0x7632));
    }
    const int rr = r & 127;
    *reinterpret_cast<uint4*>(sm_q + (r >> 7) * S::TILE + (c >> 3) * HALF + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = w;
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = ctrl->tmem;

  auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool {
    if (*abort_flag) return false;
    if (!mbar_wait(bar, parity, site)) {
      *abort_flag = 1;
      return false;
    }
    return true;
  };

  if (warp >= 12) {
    // ---------------- int8: codes to bf16 slots ----------------
    if constexpr (I8) {
      regs_dec<S::REGS_CONVERT>();
      constexpr int NL = D / 16;  // 16-byte loads of a lane: 32 rows of a warp
      const int w = warp - 12;
      const int32_t* table = p.kv.table + (size_t)blk.b * p.kv.max_pages;
      const int slot_mask = (1 << p.kv.page_shift) - 1;
      int pg[2] = {0, 0};  // pages of the warp's rows 0-15 and 16-31 in the tile being loaded
      auto look_up = [&](int j) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = k0 + j * PCH_KB + 32 * w + 16 * h;
          int page = 0;
          if (j < ntile && key < k1) {
            page = table[key >> p.kv.page_shift];
            if (page < 0 || page >= p.kv.num_pages) {
              record_error(DEV_ERR_BOUNDS, 361);
              page = 0;
            }
          }
          pg[h] = page;
        }
      };
      // row (of the warp's 32) and 16-byte chunk of load u: eight lanes read 128
      // contiguous bytes' worth of banks and write eight different chunks
      auto place = [&](int u, int& row, int& c) {
        if (D == 128) {
          c = lane & 7;
          row = 2 * ((u >> 1) * 4 + (lane >> 3)) + (((lane >> 2) & 1) ^ (u & 1));
        } else {
          c = lane & 3;
          row = u * 8 + (lane >> 2);
        }
      };
      auto load = [&](int j, const uint8_t* pool, uint4 (&buf)[NL]) {
#pragma unroll
        for (int u = 0; u < NL; ++u) {
          int row, c;
          place(u, row, c);
          const int key = k0 + j * PCH_KB + 32 * w + row;
          buf[u] = make_uint4(0, 0, 0, 0);
          if (j < ntile && key < k1)
            buf[u] = *reinterpret_cast<const uint4*>(pool + paged_row(p.kv, row < 16 ? pg[0] : pg[1], g, key & slot_mask) * D +
                                                     c * 16);
        }
      };
      auto convert = [&](int it, const uint4 (&buf)[NL]) -> bool {
        const int slot = it % S::NSLOT;
        if (it >= S::NSLOT && !__all_sync(0xffffffffu, wait(&ctrl->empty[slot], ((it / S::NSLOT) + 1) & 1, 362)))
          return false;
        uint8_t* dst = sm_slots + slot * S::TILE;
#pragma unroll
        for (int u = 0; u < NL; ++u) {
          int row, c;
          place(u, row, c);
          row += 32 * w;
          uint8_t* at = dst + (c >> 2) * HALF + row * 128;
          const uint4 x = buf[u];
          *reinterpret_cast<uint4*>(at + (((2 * (c & 3)) ^ (row & 7)) << 4)) =
              make_uint4(codes_bf2(x.x), codes_bf2(x.x >> 8), codes_bf2(x.y), codes_bf2(x.y >> 8));
          *reinterpret_cast<uint4*>(at + (((2 * (c & 3) + 1) ^ (row & 7)) << 4)) =
              make_uint4(codes_bf2(x.z), codes_bf2(x.z >> 8), codes_bf2(x.w), codes_bf2(x.w >> 8));
        }
        return true;
      };
      auto arrive = [&](int it) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctrl->full[it % S::NSLOT]);
      };
      uint4 bk[NL], bv[NL];
      look_up(0);
      load(0, p.kv.k, bk);
      for (int j = 0; j < ntile; ++j) {
        // this lane's row: its scales (0 past the part's keys)
        const int key = k0 + j * PCH_KB + 32 * w + lane;
        float ks = 0.f, vs = 0.f;
        if (key < k1) {
          const size_t row = paged_row(p.kv, lane < 16 ? pg[0] : pg[1], g, key & slot_mask);
          ks = p.kv.ks[row];
          vs = p.kv.vs[row];
        }
        load(j, p.kv.v, bv);
        if (!convert(2 * j, bk)) break;
        float* sc = sm_scale + (j % S::RING) * 256 + 32 * w + lane;
        sc[0] = ks;
        sc[128] = vs;
        arrive(2 * j);
        look_up(j + 1);
        load(j + 1, p.kv.k, bk);
        if (!convert(2 * j + 1, bv)) break;
        arrive(2 * j + 1);
      }
    }
  } else if (warp >= 8) {
    regs_dec<S::REGS_MMA>();
    if (warp == 8 && lane == 0 && ntile > 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t idesc_s = idesc_bf16_f32(128, PCH_KB);
      constexpr uint32_t idesc_o = idesc_bf16_f32(128, D) | (1u << 16);  // V: dims contiguous
      const uint32_t q0 = smem_u32(sm_q), s0 = smem_u32(sm_slots);
      auto qk = [&](int t, int j) {
        const uint32_t a = q0 + t * S::TILE, b = s0 + ((2 * j) % S::NSLOT) * S::TILE;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k >> 2) * HALF + (k & 3) * 32;
          mma_f16_ss(tbase + t * 128, smem_desc_sw128(a + off, 16, 1024), smem_desc_sw128(b + off, 16, 1024), idesc_s, k > 0);
        }
      };
      auto pv = [&](int t, int j) {
        const uint32_t b = s0 + ((2 * j + 1) % S::NSLOT) * S::TILE;
#pragma unroll
        for (int k = 0; k < PCH_KB / 16; ++k)
          mma_f16_ts(tbase + 256 + t * D, tbase + t * 128 + k * 8, smem_desc_sw128(b + k * 2048, HALF, 1024), idesc_o,
                     (j | k) > 0);
      };
      auto filled = [&](int it, int site) {
        const bool ok = wait(&ctrl->full[it % S::NSLOT], (it / S::NSLOT) & 1, site);
        tc_fence_after();
        return ok;
      };
      bool ok = filled(0, 363);
      if (ok) {
        if (n0 > 0) {
          qk(0, 0);
          tc_commit(&ctrl->s_full[0]);
        }
        if (n1 > 0) {
          qk(1, 0);
          tc_commit(&ctrl->s_full[1]);
        }
        tc_commit(&ctrl->empty[0]);
      }
      for (int j = 0; ok && j < ntile; ++j) {
        ok = filled(2 * j + 1, 364);
        bool next = false;  // K of tile j + 1 seen
        for (int t = 0; ok && t < 2; ++t) {
          const int nt = t ? n1 : n0;
          if (j < nt) {
            ok = wait(&ctrl->p_ready[t], j & 1, 365);
            if (!ok) break;
            tc_fence_after();
            pv(t, j);
          }
          if (t == (n1 > 0)) tc_commit(&ctrl->empty[(2 * j + 1) % S::NSLOT]);  // V read by its last tile
          if (j + 1 < nt) {
            if (!next) ok = filled(2 * j + 2, 366);
            if (!ok) break;
            next = true;
            qk(t, j + 1);
            tc_commit(&ctrl->s_full[t]);
          } else if (j + 1 == nt) {
            tc_commit(&ctrl->o_full[t]);
          }
        }
        if (next) tc_commit(&ctrl->empty[(2 * j + 2) % S::NSLOT]);
      }
      if (!ok) {  // let the MMAs in flight end before tensor memory is freed
        tc_commit(&ctrl->drain);
        mbar_wait(&ctrl->drain, 0, 367);
      }
    } else if (!I8 && warp == 9) {
      // ---------------- bf16: TMA loads ----------------
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
        for (int v = 0; v < 2; ++v) {
          const int it = 2 * j + v, slot = it % S::NSLOT;
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
      if (*abort_flag) {  // copies in flight land before the CTA gives its memory back
        if (tail_issued) mbar_wait(&ctrl->tail, 0, 370);
        for (int it = max(0, issued - S::NSLOT); it < issued - (tail_issued ? 1 : 0); ++it)
          mbar_wait(&ctrl->full[it % S::NSLOT], (it / S::NSLOT) & 1, 370);
      }
    }
  } else {
    // ---------------- softmax: a thread owns a row ----------------
    regs_inc<S::REGS_SOFTMAX>();
    const int t = warp >> 2, r = t * 128 + (warp & 3) * 32 + lane;
    const int nt = t ? n1 : n0;
    const bool live = r < blk.nrows;
    const bool warp_live = r - lane < blk.nrows;
    const int row = blk.row0 + r, tok = row / p.G;
    const int lim = live ? blk.past + tok + 1 : INT_MAX;
    const int lim_min = __reduce_min_sync(0xffffffffu, lim);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tbase + lanes + t * 128, to = tbase + lanes + 256 + t * D;
    const uint64_t scale2 = f2_splat(p.scale_log2);
    float m = -INFINITY;
    uint64_t l2[2] = {0, 0};
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      ok = wait(&ctrl->s_full[t], j & 1, 371);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (warp_live) {
        uint32_t s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, s + 32 * c);
        tmem_wait_ld();
        const float* sc = sm_scale + (j % S::RING) * 256;
        if (I8) {
#pragma unroll
          for (int c = 0; c < 128; c += 4) {
            const float4 k = *reinterpret_cast<const float4*>(sc + c);
            s[c] = __float_as_uint(__uint_as_float(s[c]) * k.x);
            s[c + 1] = __float_as_uint(__uint_as_float(s[c + 1]) * k.y);
            s[c + 2] = __float_as_uint(__uint_as_float(s[c + 2]) * k.z);
            s[c + 3] = __float_as_uint(__uint_as_float(s[c + 3]) * k.w);
          }
        }
        const int base = k0 + j * PCH_KB;
        if (base + PCH_KB > min(lim_min, k1)) {
          const int see = min(lim, k1) - base;
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= see) s[c] = 0xff800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 128; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(s[c]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
        if (j == 0) {
          m = top;
        } else if (__any_sync(0xffffffffu, top > m + 8.f)) {
          const float mn = fmaxf(m, top);
          const float f = mn == -INFINITY ? 1.f : ex2(m - mn);
          m = mn;
          const uint64_t f2 = f2_splat(f);
          l2[0] = f2_mul(l2[0], f2);
          l2[1] = f2_mul(l2[1], f2);
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
        const uint64_t ref2 = f2_splat(m == -INFINITY ? 0.f : -m);
#pragma unroll
        for (int c = 0; c < 128; c += 32) {
          uint32_t pw[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            uint32_t a, b;
            f2_split(f2_fma(f2_make(s[c + 2 * e], s[c + 2 * e + 1]), scale2, ref2), a, b);
            float x = ex2(__uint_as_float(a)), y = ex2(__uint_as_float(b));
            l2[e & 1] = f2_add(l2[e & 1], f2_make(__float_as_uint(x), __float_as_uint(y)));
            if (I8) {
              const float2 v = *reinterpret_cast<const float2*>(sc + 128 + c + 2 * e);
              // a masked key's scale may be anything
              x = x == 0.f ? 0.f : x * v.x;
              y = y == 0.f ? 0.f : y * v.y;
            }
            pw[e] = bf2_of(x, y);
          }
          tmem_st16(ts + c / 2, pw);
        }
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctrl->p_ready[t]);
    }
    if (ok && nt > 0) ok = __all_sync(0xffffffffu, wait(&ctrl->o_full[t], 0, 372));
    if (ok && warp_live) {
      tc_fence_after();
      uint32_t a, b, c2, d2;
      f2_split(l2[0], a, b);
      f2_split(l2[1], c2, d2);
      const float l = (__uint_as_float(a) + __uint_as_float(b)) + (__uint_as_float(c2) + __uint_as_float(d2));
      const float inv = m == -INFINITY ? 0.f : 1.f / l;
      const size_t pr = (((size_t)sp * p.blocks + bx) * p.kv.n_kv + g) * PCH_R + r;
      if (live && nparts > 1) p.part_ml[pr] = make_float2(m, l);
      uint16_t* dst = p.out + ((size_t)(blk.tok0 + tok) * p.n_heads + g * p.G + row - tok * p.G) * D;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
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
              w[k] = m == -INFINITY ? 0u
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
