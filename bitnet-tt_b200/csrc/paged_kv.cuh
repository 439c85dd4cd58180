// Paged KV cache: what its kernels share, and the kernels that write and read it.
//
// A pool of pages [num_pages][n_kv_heads][page_size][head_dim] holds keys (and
// another values) as bf16, or as int8 with one fp32 scale per (page, KV head,
// row); the value of a code is code * scale.  Row `pos` of sequence b is row
// pos % page_size of page block_table[b][pos / page_size].
//
// Page ids, offsets and lengths are device data, so the kernels check them: a
// bad one is recorded in the device status word (DEV_ERR_BOUNDS) and the access
// is skipped.
#pragma once
#include "common.cuh"

namespace bitnet {

struct PagedKV {
  uint8_t* k;          // pages of keys (bf16 or int8)
  uint8_t* v;
  float* ks;           // int8: scales [num_pages][n_kv][page_size]
  float* vs;
  int num_pages, page_shift, n_kv;
  const int32_t* table;  // [B][max_pages]
  int max_pages;
};

// Row index (in units of head_dim elements) of row `slot` of KV head g in `page`.
__device__ __forceinline__ size_t paged_row(const PagedKV& c, int page, int g, int slot) {
  return ((((size_t)page * c.n_kv + g) << c.page_shift) + slot);
}

// The last b in 0 .. B-1 with cu[b] <= row, found by a whole warp: each round
// narrows the range 32 times (two rounds up to 1024 sequences).  An empty
// sequence is never the answer for a row that some sequence holds.
__device__ __forceinline__ int warp_find_seq(const int32_t* cu, int B, int row, int lane) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int idx = lo + (lane + 1) * step;
    const unsigned le = __ballot_sync(0xffffffffu, idx < hi && cu[idx] <= row);
    lo += __popc(le) * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

__device__ __forceinline__ uint32_t bf2_of(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void unpack_bf8(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack_bf8(const float (&x)[8]) {
  return make_uint4(bf2_of(x[0], x[1]), bf2_of(x[2], x[3]), bf2_of(x[4], x[5]), bf2_of(x[6], x[7]));
}

// Four codes of a word as fp32 values, and four fp32 values of at most 127.49 as
// codes (half to even), without the conversion unit, which handles 16 values a
// cycle and SM: fp32 0x4B0000uu is 2^23 + u, and v + 1.5 * 2^23 holds rint(v) in its
// low byte.
__device__ __forceinline__ void codes_to_f32(uint32_t w, float* x) {
  w ^= 0x80808080u;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __fsub_rn(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 + e)), 8388736.f);
}
__device__ __forceinline__ uint32_t codes_of_f32(float a, float b, float c, float d) {
  const uint32_t m0 = __float_as_uint(__fadd_rn(a, 12582912.f)), m1 = __float_as_uint(__fadd_rn(b, 12582912.f));
  const uint32_t m2 = __float_as_uint(__fadd_rn(c, 12582912.f)), m3 = __float_as_uint(__fadd_rn(d, 12582912.f));
  return __byte_perm(__byte_perm(m0, m1, 0x0040), __byte_perm(m2, m3, 0x0040), 0x5410);
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// For pair j < rot/2 of a query or key head, (a, b) = dims (j, j + rot/2), or
// (2j, 2j + 1) when interleaved:
//     a' = a cos[pos][j] - b sin[pos][j],   b' = b cos[pos][j] + a sin[pos][j]
// in fp32, each product and sum rounded on its own (so an int8 code is a
// function of the inputs alone, not of how the compiler fuses), and the dims
// from rot on copied.  A value is rounded once, to bf16 or to its int8 code; with
// `stepwise` every product and sum is rounded to bf16 as well, which is what the
// bf16 model code and the contiguous cache's kernels do: the rows are then those
// kernels' bit for bit.
//     int8: top = max(max_d |row|, 1e-5), scale = top / 127, code = rint(row * (127 / top)),
// the floor of the framework's activation quantiser.  A row with an infinity or
// a NaN gets the scale NaN (its values read back as NaN).
//
// Bound: memory.  D/16 lanes take one head of one token, each the two 16-byte
// chunks that hold eight pairs (or two chunks of the dims that only move), so a
// rotation needs no shuffle and reads each table entry once; the row's maximum
// is a short shuffle tree.  In bf16 two heads a lane are loaded before the first is
// worked on (one in int8, whose work needs the registers); at 48 registers, for five
// CTAs an SM, that costs 56 to 60 bytes of spills.  Rows are loaded behind the barrier
// after the look-ups, and table entries again for each head.  B200: 32 x 512 tokens,
// 20 + 2 x 5 heads of 128, 48.1 us, 5.2 TB/s; stepwise, whose roundings are four more
// a value, 66.4 us.
struct PagedAppendParams {
  PagedKV kv;
  const int32_t* cu;       // [B + 1] token offsets
  const int32_t* kv_lens;  // [B] keys including the new tokens
  int B, tokens;
  const uint16_t* qkv;
  int ld_qkv, n_heads;
  const void* cos;         // [rope_len][rot / 2], bf16 or fp32
  const void* sin;
  int rope_len, rot, interleaved, stepwise;
  uint16_t* q_out;         // [tokens][n_heads * D]
  int tok_per_cta;         // 1 .. 8
};

constexpr int PKV_THREADS = 256;

template <bool F32>
__device__ __forceinline__ void rope_entries8(const void* t, size_t i, float (&x)[8]) {  // i % 8 == 0
  if (F32) {
    const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(t) + i);
    const float4 b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(t) + i + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    unpack_bf8(*reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(t) + i), x);
  }
}

// One rotated pair.
__device__ __forceinline__ void rotate_pair(float& a, float& b, float c, float s, bool stepwise) {
  const float ac = __fmul_rn(a, c), bs = __fmul_rn(-b, s), bc = __fmul_rn(b, c), as = __fmul_rn(a, s);
  if (stepwise) {
    a = round_bf16(__fadd_rn(round_bf16(ac), round_bf16(bs)));
    b = round_bf16(__fadd_rn(round_bf16(bc), round_bf16(as)));
  } else {
    a = __fadd_rn(ac, bs);
    b = __fadd_rn(bc, as);
  }
}

// The chunks (of 8 dims) that lane l of a head takes: c0 and c1 hold the pairs
// (d, d + rot / 2) of half layouts; adjacent pairs lie within a chunk.
__device__ __forceinline__ void append_chunks(int l, int rot, bool interleaved, int& c0, int& c1, bool& turns) {
  const int h = rot >> 4;  // lanes that turn
  turns = l < h;
  c0 = turns && !interleaved ? l : 2 * l;
  c1 = turns && !interleaved ? l + h : 2 * l + 1;
}

template <int D, bool I8, bool F32>
__global__ void __launch_bounds__(PKV_THREADS, 5) paged_append_kernel(const PagedAppendParams p) {
  constexpr int LPH = D / 16;                 // lanes of one head
  constexpr int GROUPS = PKV_THREADS / LPH;   // heads at once
  constexpr int U = I8 ? 1 : 2;               // heads of a lane in flight
  __shared__ int s_pos[8], s_page[8];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tok0 = blockIdx.x * p.tok_per_cta;
  const int ntok = min(p.tok_per_cta, p.tokens - tok0);
  if (warp < ntok) {
    const int tok = tok0 + warp;
    const int b = warp_find_seq(p.cu, p.B, tok, lane);
    if (lane == 0) {
      int pos = -1, page = -1;
      const int lo = p.cu[b], hi = p.cu[b + 1];
      if (tok >= lo && tok < hi) {  // else a row that belongs to no sequence: left alone
        pos = p.kv_lens[b] - (hi - lo) + (tok - lo);
        const int pi = pos >> p.kv.page_shift;
        if (pos < 0 || pos >= p.rope_len || pi >= p.kv.max_pages) {
          record_error(DEV_ERR_BOUNDS, 340);
          pos = -1;
        } else {
          page = p.kv.table[(size_t)b * p.kv.max_pages + pi];
          if (page < 0 || page >= p.kv.num_pages) {
            record_error(DEV_ERR_BOUNDS, 341);
            pos = -1;
          }
        }
      }
      s_pos[warp] = pos;
      s_page[warp] = page;
    }
  }
  __syncthreads();
  const int heads = p.n_heads + 2 * p.kv.n_kv, items = ntok * heads;
  int c0, c1;
  bool turns;
  append_chunks(tid % LPH, p.rot, p.interleaved, c0, c1, turns);
  for (int it0 = tid / LPH; it0 - tid / LPH < items; it0 += U * GROUPS) {
    uint4 w0[U], w1[U];
    int tk[U], hd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int it = it0 + u * GROUPS;
      const int t = it < items ? it / heads : 0;
      hd[u] = it - t * heads;
      tk[u] = it < items && s_pos[t] >= 0 ? t : -1;
      w0[u] = w1[u] = make_uint4(0, 0, 0, 0);
      if (tk[u] >= 0) {
        const uint16_t* src = p.qkv + (size_t)(tok0 + t) * p.ld_qkv + hd[u] * D;
        w0[u] = *reinterpret_cast<const uint4*>(src + c0 * 8);
        w1[u] = *reinterpret_cast<const uint4*>(src + c1 * 8);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = max(tk[u], 0), hh = hd[u], pos = s_pos[t];
      const bool live = tk[u] >= 0, is_q = hh < p.n_heads, is_v = hh >= p.n_heads + p.kv.n_kv;
      float x[8], y[8];
      unpack_bf8(w0[u], x);
      unpack_bf8(w1[u], y);
      if (live && turns && !is_v) {
        const size_t row = (size_t)pos * (p.rot >> 1);
        float c[8], s[8];
        rope_entries8<F32>(p.cos, row + (tid % LPH) * 8, c);
        rope_entries8<F32>(p.sin, row + (tid % LPH) * 8, s);
        if (p.interleaved) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            rotate_pair(x[2 * e], x[2 * e + 1], c[e], s[e], p.stepwise);
            rotate_pair(y[2 * e], y[2 * e + 1], c[4 + e], s[4 + e], p.stepwise);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) rotate_pair(x[e], y[e], c[e], s[e], p.stepwise);
        }
      }
      const int g = is_q ? 0 : (is_v ? hh - p.n_heads - p.kv.n_kv : hh - p.n_heads);
      const size_t row = live ? paged_row(p.kv, s_page[t], g, pos & ((1 << p.kv.page_shift) - 1)) : 0;
      uint8_t* pool = is_v ? p.kv.v : p.kv.k;
      if (I8 && __any_sync(0xffffffffu, live && !is_q)) {
        uint32_t top = 0;  // the largest |x| by its bits: a NaN or an infinity wins
#pragma unroll
        for (int e = 0; e < 8; ++e)
          top = max(top, max(__float_as_uint(x[e]) & 0x7fffffffu, __float_as_uint(y[e]) & 0x7fffffffu));
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (live && !is_q) {
          const bool finite = top < 0x7f800000u;
          const float amax = fmaxf(__uint_as_float(top), 1e-5f), inv = __fdiv_rn(127.f, amax);
          uint32_t q[4];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(x[e], inv), y[e] = __fmul_rn(y[e], inv);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            q[e] = codes_of_f32(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
            q[2 + e] = codes_of_f32(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
          }
          if (!finite) q[0] = q[1] = q[2] = q[3] = 0;
          *reinterpret_cast<uint2*>(pool + row * D + c0 * 8) = make_uint2(q[0], q[1]);
          *reinterpret_cast<uint2*>(pool + row * D + c1 * 8) = make_uint2(q[2], q[3]);
          if (tid % LPH == 0)
            (is_v ? p.kv.vs : p.kv.ks)[row] = finite ? __fdiv_rn(amax, 127.f) : __uint_as_float(0x7fc00000u);
        }
      }
      if (live && (is_q || !I8)) {
        uint16_t* dst = is_q ? p.q_out + ((size_t)(tok0 + t) * p.n_heads + hh) * D : reinterpret_cast<uint16_t*>(pool) + row * D;
        *reinterpret_cast<uint4*>(dst + c0 * 8) = pack_bf8(x);
        *reinterpret_cast<uint4*>(dst + c1 * 8) = pack_bf8(y);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// read
// ---------------------------------------------------------------------------
// Row r of sequence b's packed rows (cu[b] .. cu[b + 1] - 1) is cache row
// starts[b] + r - cu[b]; k_out / v_out are bf16 [rows][n_kv][D].  int8: the value
// bf16(code * scale), rounded once.  Bound: memory, one pass; a lane moves 16 bytes
// of two rows at a time, neighbours in a page side by side.  Eight rows a CTA and
// six CTAs an SM: the look-ups before the first load hide behind other CTAs (16
// rows and four loads in flight took 31.5 us where this takes 29.0, 4.6 TB/s, for 16
// ragged int8 contexts of up to 4096 rows).
struct PagedReadParams {
  PagedKV kv;
  const int32_t* cu;
  const int32_t* starts;  // nullable: 0
  int B, rows;
  uint16_t* k_out;
  uint16_t* v_out;
};
constexpr int PKV_READ_ROWS = 8;

template <int D, bool I8>
__global__ void __launch_bounds__(PKV_THREADS, 6) paged_read_kernel(const PagedReadParams p) {
  constexpr int LPH = D / (I8 ? 16 : 8);  // lanes of a row, 16 bytes each
  constexpr int GROUPS = PKV_THREADS / LPH;
  constexpr int U = 2;
  __shared__ int s_slot[PKV_READ_ROWS], s_page[PKV_READ_ROWS];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31;
  const int row0 = blockIdx.x * PKV_READ_ROWS, nrow = min(PKV_READ_ROWS, p.rows - row0);
  for (int i = tid >> 5; i < nrow; i += PKV_THREADS / 32) {
    const int r = row0 + i;
    const int b = warp_find_seq(p.cu, p.B, r, lane);
    if (lane == 0) {
      int page = -1, slot = 0;
      if (r >= p.cu[b] && r < p.cu[b + 1]) {
        const long long pos = (long long)(p.starts ? p.starts[b] : 0) + (r - p.cu[b]);
        const long long pi = pos >> p.kv.page_shift;
        if (pos < 0 || pi >= p.kv.max_pages) {
          record_error(DEV_ERR_BOUNDS, 342);
        } else {
          slot = (int)pos & ((1 << p.kv.page_shift) - 1);
          page = p.kv.table[(size_t)b * p.kv.max_pages + pi];
          if (page < 0 || page >= p.kv.num_pages) {
            record_error(DEV_ERR_BOUNDS, 343);
            page = -1;
          }
        }
      }
      s_page[i] = page;
      s_slot[i] = slot;
    }
  }
  __syncthreads();
  const int per_row = 2 * p.kv.n_kv, items = nrow * per_row;
  const int l = tid % LPH;
  for (int it0 = tid / LPH; it0 < items; it0 += U * GROUPS) {
    uint4 w[U];
    float sc[U];
    uint16_t* dst[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int it = it0 + u * GROUPS;
      const int h = it < items ? it / nrow : 0, t = it - h * nrow;  // neighbours in a page side by side
      dst[u] = nullptr;
      if (it < items && s_page[t] >= 0) {
        const bool is_v = h >= p.kv.n_kv;
        const int g = is_v ? h - p.kv.n_kv : h;
        const size_t row = paged_row(p.kv, s_page[t], g, s_slot[t]);
        w[u] = *reinterpret_cast<const uint4*>((is_v ? p.kv.v : p.kv.k) + row * (I8 ? D : 2 * D) + l * 16);
        if (I8) sc[u] = (is_v ? p.kv.vs : p.kv.ks)[row];
        dst[u] = (is_v ? p.v_out : p.k_out) + ((size_t)(row0 + t) * p.kv.n_kv + g) * D;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (dst[u] == nullptr) continue;
      if (I8) {
        const uint32_t c[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[8];
          codes_to_f32(c[2 * h], x);
          codes_to_f32(c[2 * h + 1], x + 4);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(x[e], sc[u]);
          *reinterpret_cast<uint4*>(dst[u] + l * 16 + h * 8) = pack_bf8(x);
        }
      } else {
        *reinterpret_cast<uint4*>(dst[u] + l * 8) = w[u];
      }
    }
  }
}

}  // namespace bitnet
