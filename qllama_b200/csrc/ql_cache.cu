// ql_cache.cu -- kernels around the paged KV cache for B200 (sm_100a): appending and
// reading the rows of several sequences, and choosing the blocks of a long cache that a
// query attends to.
#include <math_constants.h>

#include <algorithm>

#include "ql_append.cuh"
#include "ql_device.cuh"
#include "ql_kernels.cuh"

namespace ql {

namespace {

// The sequence that token r belongs to (empty ones are passed over).
__device__ __forceinline__ int ragged_seq(const RaggedTable& t, int batch, int r) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= r) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Eight consecutive values as they are in memory, and as f32.
struct Raw8 {
  uint4 w[2];  // the second for f32 only
};

__device__ __forceinline__ Raw8 load_raw8(const void* base, size_t i, int dt, bool vec) {
  Raw8 r;
  if (vec && dt == kF32) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + i);
    r.w[0] = p[0];
    r.w[1] = p[1];
  } else if (vec) {
    r.w[0] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
  } else if (dt == kF32) {
    const uint32_t* p = static_cast<const uint32_t*>(base) + i;
    r.w[0] = make_uint4(p[0], p[1], p[2], p[3]);
    r.w[1] = make_uint4(p[4], p[5], p[6], p[7]);
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(base) + i;
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = p[2 * k] | static_cast<uint32_t>(p[2 * k + 1]) << 16;
    r.w[0] = make_uint4(x[0], x[1], x[2], x[3]);
  }
  return r;
}

__device__ __forceinline__ void floats_of(const Raw8& r, int dt, float (&x)[8]) {
  if (dt == kF32) {
    const uint32_t in[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w,
                            r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(in[k]);
    return;
  }
  const uint32_t in[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = dt == kF16 ? __half22float2(*reinterpret_cast<const __half2*>(&in[k]))
                                : make_float2(__uint_as_float(in[k] << 16),
                                              __uint_as_float(in[k] & 0xffff0000u));
    x[2 * k] = f.x, x[2 * k + 1] = f.y;
  }
}

// Where one thread's dims d .. d + 7 of a position lie in the cache, for KV head 0, and the bytes
// from head to head: computed once for all heads.
struct RowPlace {
  uint8_t *k, *v, *v2, *ks, *vs;  // v2: of dims d + 4 .. (Q4_0); ks, vs: the block's scale
  size_t step, scale_step;
};

template <int KIND>
__device__ __forceinline__ RowPlace row_place(const CacheView& c, int page, int pos, int d) {
  RowPlace p;
  const int off = pos % c.page;
  const size_t row = static_cast<size_t>(page) * c.hkv * c.page + off;
  if constexpr (KIND == kQ4_0) {
    const Q4Record rec{c.hd};
    const int per = c.page / kTile, nb = c.hd / 32, at = off % kTile;
    uint8_t* base = static_cast<uint8_t*>(c.k) +
                    (static_cast<size_t>(page) * c.hkv * per + off / kTile) * rec.bytes();
    p.k = base + q4_k_byte(at, d, nb);
    p.v = base + rec.v_codes() + q4_v_byte(at, d, nb);
    p.v2 = base + rec.v_codes() + q4_v_byte(at, d + 4, nb);
    p.ks = base + rec.k_scales() + 2 * q4_k_scale(at, d / 32, nb);
    p.vs = base + rec.v_scales() + 2 * q4_v_scale(at, d / 32, nb);
    p.step = p.scale_step = per * rec.bytes();
  } else {
    const size_t size = KIND == kQ8_0 ? 1 : c.dtype == kF32 ? 4 : 2;
    p.k = static_cast<uint8_t*>(c.k) + (row * c.hd + d) * size;
    p.v = static_cast<uint8_t*>(c.v) + (row * c.hd + d) * size;
    p.v2 = nullptr;
    p.step = static_cast<size_t>(c.page) * c.hd * size;
    p.ks = KIND == kQ8_0 ? reinterpret_cast<uint8_t*>(c.k_scale + row * (c.hd / 32) + d / 32) : nullptr;
    p.vs = KIND == kQ8_0 ? reinterpret_cast<uint8_t*>(c.v_scale + row * (c.hd / 32) + d / 32) : nullptr;
    p.scale_step = static_cast<size_t>(c.page) * (c.hd / 32) * 2;
  }
  return p;
}

// Writes eight values of KV head h; four neighbouring lanes hold a block of 32.  KIND: kQ8_0,
// kQ4_0, or kF32 for the types that need no block.
template <int KIND>
__device__ __forceinline__ void store_cache8(const RowPlace& p, int dtype, int h, bool v,
                                             const float (&x)[8], bool live, uint32_t lanes) {
  uint8_t* at = (v ? p.v : p.k) + h * p.step;
  if constexpr (KIND == kF32) {
    if (live) store8(at, 0, dtype, x, true);
    return;
  }
  const int lane = threadIdx.x & 31;
  uint16_t* scale_at = reinterpret_cast<uint16_t*>((v ? p.vs : p.ks) + h * p.scale_step);
  if constexpr (KIND == kQ8_0) {
    // q8_0_pair's rule, but for the rounding of d: a product, not a division
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(x[k]));
    amax = fmaxf(amax, __shfl_xor_sync(lanes, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(lanes, amax, 2));
    const float s = amax * (1.0f / 127.0f), id = s != 0.0f ? 1.0f / s : 0.0f;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float r = roundf(x[k] * id);
      w[k / 4] |= (static_cast<uint32_t>(r == r ? static_cast<int>(r) : 0) & 0xffu) << (8 * (k & 3));
    }
    if (live) {
      *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
      if ((lane & 3) == 0) *scale_at = __half_as_ushort(__float2half_rn(s));
    }
    return;
  }
  // Q4_0: the value of largest magnitude, of equal ones the first (in the lower lane)
  float m = x[0];
  bool finite = fabsf(x[0]) < CUDART_INF_F;
#pragma unroll
  for (int k = 1; k < 8; ++k) {
    if (fabsf(x[k]) > fabsf(m)) m = x[k];
    finite = finite && fabsf(x[k]) < CUDART_INF_F;
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const float w = __shfl_xor_sync(lanes, m, o);
    if (fabsf(w) > fabsf(m) || (fabsf(w) == fabsf(m) && (lane & o))) m = w;
  }
  finite = (__ballot_sync(lanes, !finite) >> (lane & 28) & 15u) == 0;
  const uint16_t scale = q4_scale(m, finite);
  const float s = __half2float(__ushort_as_half(scale));
  const uint32_t w = scale == kHalfNan || s == 0.f ? 0x88888888u : q4_codes8(x, s, q4_inverse(s));
  if (!live) return;
  if (v) {  // two lanes' places
    *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(w);
    *reinterpret_cast<uint16_t*>(p.v2 + h * p.step) = static_cast<uint16_t>(w >> 16);
  } else {
    *reinterpret_cast<uint32_t*>(at) = w;
  }
  if ((lane & 3) == 0) *scale_at = scale;
}

// The converse, in two steps so that several rows' loads are under way together: eight values of
// KV head h as they lie there (a word or two of codes, the scale behind them), and as f32.
template <int KIND>
__device__ __forceinline__ Raw8 load_cache8(const RowPlace& p, int dtype, int h, bool v) {
  const uint8_t* at = (v ? p.v : p.k) + h * p.step;
  if constexpr (KIND == kF32) return load_raw8(at, 0, dtype, true);
  Raw8 r;
  r.w[0].z = *reinterpret_cast<const uint16_t*>((v ? p.vs : p.ks) + h * p.scale_step);
  if constexpr (KIND == kQ8_0) {
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    r.w[0].x = w.x, r.w[0].y = w.y;
  } else {
    r.w[0].x = v ? *reinterpret_cast<const uint16_t*>(at) |
                       static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p.v2 + h * p.step)) << 16
                 : *reinterpret_cast<const uint32_t*>(at);
  }
  return r;
}

template <int KIND>
__device__ __forceinline__ void cache8_values(const Raw8& r, int dtype, float (&x)[8]) {
  if constexpr (KIND == kF32) {
    floats_of(r, dtype, x);
    return;
  }
  const float s = __half2float(__ushort_as_half(static_cast<uint16_t>(r.w[0].z)));
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (KIND == kQ8_0)
      x[k] = s * static_cast<float>(
                     static_cast<int8_t>((k < 4 ? r.w[0].x : r.w[0].y) >> (8 * (k & 3))));
    else
      x[k] = s * static_cast<float>(static_cast<int>(r.w[0].x >> (4 * k) & 15u) - 8);
  }
}

// The page of a position, -1 (and the status raised) if the table's entry is outside the pool.
__device__ __forceinline__ int page_of(const CacheView& c, int seq, int pos, uint32_t* status) {
  const int page = c.block_table[static_cast<size_t>(seq) * c.pages_per_seq + pos / c.page];
  if (page >= 0 && page < c.num_pages) return page;
  if (status) atomicOr(status, kStatusBadPage);
  return -1;
}

constexpr int kAtOnce = 4;  // rows whose loads a thread has under way together

}  // namespace

// ---------------------------------------------------------------- append --
// A row of HD values takes HD / 8 lanes, eight values each: 16-byte loads, and four lanes a
// block of 32.  The block's groups of lanes have a token each and take the same a.rows_each rows
// of them (of the query, key and value heads in that order; blockIdx.y says which), kAtOnce at a
// time; the position's angles are fetched once for all.  Neighbouring tokens stand in one warp,
// whose stores of V codes then fill whole words.
// IN: the input type, with every tensor 16-byte aligned; -1: read from the arguments, in any
// place.  KIND: as store_cache8's.
// Bound by the f64 rotation (six operations and four conversions a pair, the conversions at an
// eighth of the rate of f32 arithmetic) and, to Q4_0, the quantiser's instructions; the bytes
// are about half of it: 6044 packed tokens of 32 + 2 x 8 heads in bf16 take 30 us (130 MB), 8192
// to Q4_0 52 us (177 MB).
template <int HD, int IN, int KIND>
__global__ void __launch_bounds__(256, 3) ragged_append_kernel(const __grid_constant__ RaggedAppendArgs a) {
  constexpr int kLanes = HD / 8;
  const CacheView& c = a.cache;
  const int in_dt = IN >= 0 ? IN : a.in_dtype;
  const int r = static_cast<int>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  if (r >= a.rows.first[a.batch]) return;
  const uint32_t lanes =  // of this group, for its shuffles
      ((1u << kLanes) - 1) << (threadIdx.x & 31 & ~(kLanes - 1));
  const int heads = a.hq + 2 * c.hkv;
  const int h0 = blockIdx.y * a.rows_each, h1 = min(h0 + a.rows_each, heads);
  const int d = threadIdx.x % kLanes * 8;
  const int b = ragged_seq(a.rows, a.batch, r);
  const int pos = a.rows.start[b] + r - a.rows.first[b];
  double2 cs[4];
  const bool turn = a.rope && h0 < a.hq + c.hkv;
  if (turn) {
    const double2* p = a.rope + static_cast<size_t>(pos) * (HD / 2) + d / 2;
#pragma unroll
    for (int k = 0; k < 4; ++k) cs[k] = p[k];
  }
  int page = 0;
  RowPlace place{};
  if (h1 > a.hq) {
    page = page_of(c, a.rows.seq[b], pos, a.status);
    place = row_place<KIND>(c, max(page, 0), pos, d);
  }
  const int size = in_dt == kF32 ? 4 : 2, out_size = a.q_out_dtype == kF32 ? 4 : 2;
  const size_t tok = static_cast<size_t>(r);
  const uint8_t* q_at = static_cast<const uint8_t*>(a.q) + (tok * a.q_stride + d) * size;
  const uint8_t* k_at = static_cast<const uint8_t*>(a.k) + (tok * a.k_stride + d) * size;
  const uint8_t* v_at = static_cast<const uint8_t*>(a.v) + (tok * a.v_stride + d) * size;
  uint8_t* out_at = static_cast<uint8_t*>(a.q_out) + (tok * a.hq * HD + d) * out_size;
  for (int g0 = h0; g0 < h1; g0 += kAtOnce) {
    Raw8 raw[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int h = min(g0 + i, h1 - 1);
      const bool q = h < a.hq, k = h < a.hq + c.hkv;
      const uint8_t* at = q ? q_at : k ? k_at : v_at;
      const int in_row = h - (q ? 0 : k ? a.hq : a.hq + c.hkv);
      raw[i] = load_raw8(at + in_row * HD * size, 0, in_dt,
                         IN >= 0 || a.vec >> (q ? 0 : k ? 1 : 2) & 1);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int h = g0 + i;
      if (h >= h1) break;
      float x[8];
      floats_of(raw[i], in_dt, x);
      if (turn && h < a.hq + c.hkv) {
#pragma unroll
        for (int k = 0; k < 4; ++k) rope_pair(x[2 * k], x[2 * k + 1], cs[k], x[2 * k], x[2 * k + 1]);
      }
      if (h < a.hq) {
        store8(out_at + h * HD * out_size, 0, a.q_out_dtype, x, IN >= 0 || (a.vec & 8) != 0);
      } else {
        const bool v = h >= a.hq + c.hkv;
        store_cache8<KIND>(place, c.dtype, h - a.hq - (v ? c.hkv : 0), v, x, page >= 0, lanes);
      }
    }
  }
}

// Any head size: one warp per query row, or per key and value row of a KV head.
__global__ void __launch_bounds__(128) ragged_append_any_kernel(const __grid_constant__ RaggedAppendArgs a) {
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const CacheView& c = a.cache;
  const int heads = a.hq + c.hkv, hd = c.hd;
  const int64_t r64 = warp / heads;
  if (r64 >= a.rows.first[a.batch]) return;
  const int r = static_cast<int>(r64), h = static_cast<int>(warp - r64 * heads);
  const int b = ragged_seq(a.rows, a.batch, r);
  const int pos = a.rows.start[b] + r - a.rows.first[b];
  const double2* rope = a.rope ? a.rope + static_cast<size_t>(pos) * (hd / 2) : nullptr;
  if (h < a.hq) {
    const size_t in = static_cast<size_t>(r) * a.q_stride + static_cast<size_t>(h) * hd;
    const size_t out = (static_cast<size_t>(r) * a.hq + h) * hd;
    for (int p = lane; p < hd / 2; p += 32) {
      float y0 = load_elem(a.q, in + 2 * p, a.in_dtype);
      float y1 = load_elem(a.q, in + 2 * p + 1, a.in_dtype);
      if (rope) rope_pair(y0, y1, rope[p], y0, y1);
      store_elem(a.q_out, out + 2 * p, a.q_out_dtype, y0);
      store_elem(a.q_out, out + 2 * p + 1, a.q_out_dtype, y1);
    }
    return;
  }
  const int kvh = h - a.hq;
  bool ok;
  const int64_t dst = cache_row(c, a.rows.seq[b], pos, kvh, a.status, ok);
  if (!ok) return;
  append_row<true>(a.k, a.v, a.in_dtype, static_cast<size_t>(r) * a.k_stride + static_cast<size_t>(kvh) * hd,
                   static_cast<size_t>(r) * a.v_stride + static_cast<size_t>(kvh) * hd, rope, c, dst, lane);
}

namespace {

using AppendFn = void (*)(const RaggedAppendArgs);

template <int HD, int IN>
AppendFn append_form(int dtype) {
  return dtype == kQ4_0   ? ragged_append_kernel<HD, IN, kQ4_0>
         : dtype == kQ8_0 ? ragged_append_kernel<HD, IN, kQ8_0>
                          : ragged_append_kernel<HD, IN, kF32>;
}

template <int HD>
AppendFn append_form(int in_dt, int dtype) {
  return in_dt == kF32    ? append_form<HD, kF32>(dtype)
         : in_dt == kF16  ? append_form<HD, kF16>(dtype)
         : in_dt == kBF16 ? append_form<HD, kBF16>(dtype)
                          : append_form<HD, -1>(dtype);
}

}  // namespace

cudaError_t launch_ragged_append(const RaggedAppendArgs& a_in, cudaStream_t s) {
  RaggedAppendArgs a = a_in;
  const int64_t tokens = a.rows.first[a.batch];
  if (tokens == 0) return cudaSuccess;
  const int hd = a.cache.hd, heads = a.hq + 2 * a.cache.hkv;
  // 16-byte accesses where the base and every row allow them
  const int64_t per = a.in_dtype == kF32 ? 4 : 8;
  auto fits = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  a.vec = (fits(a.q) && a.q_stride % per == 0 ? 1 : 0) | (fits(a.k) && a.k_stride % per == 0 ? 2 : 0) |
          (fits(a.v) && a.v_stride % per == 0 ? 4 : 0) | (fits(a.q_out) ? 8 : 0);
  if (hd != 64 && hd != 128) {
    const int64_t threads = tokens * (a.hq + a.cache.hkv) * 32;
    ragged_append_any_kernel<<<static_cast<unsigned>((threads + 127) / 128), 128, 0, s>>>(a);
    return cudaGetLastError();
  }
  // Rows of a thread: kAtOnce, or twice as many where the blocks are many waves anyway (the angles
  // are then read half as often).
  const int64_t blocks = (tokens * (hd / 8) + 255) / 256;
  const int chunks = (heads + kAtOnce - 1) / kAtOnce;
  a.rows_each = blocks * chunks > 4096 ? 2 * kAtOnce : kAtOnce;
  const int in = a.vec == 15 ? a.in_dtype : -1;
  const AppendFn k = hd == 64 ? append_form<64>(in, a.cache.dtype) : append_form<128>(in, a.cache.dtype);
  k<<<dim3(static_cast<unsigned>(blocks), (heads + a.rows_each - 1) / a.rows_each), 256, 0, s>>>(a);
  return cudaGetLastError();
}

// ------------------------------------------------------------------ read --
// As the append: HD / 8 lanes have a token and read kAtOnce KV heads of it (blockIdx.y says
// which), K and V.
template <int HD, int KIND>
__global__ void __launch_bounds__(256) ragged_read_kernel(const __grid_constant__ RaggedReadArgs a) {
  constexpr int kLanes = HD / 8;
  const CacheView& c = a.cache;
  const int r = static_cast<int>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  if (r >= a.rows.first[a.batch]) return;
  const int d = threadIdx.x % kLanes * 8;
  const int b = ragged_seq(a.rows, a.batch, r);
  const int pos = a.rows.start[b] + r - a.rows.first[b];
  const int page = page_of(c, a.rows.seq[b], pos, a.status);
  const RowPlace place = row_place<KIND>(c, max(page, 0), pos, d);
  const int h0 = blockIdx.y * kAtOnce;
  Raw8 raw[kAtOnce][2];
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
    for (int v = 0; v < 2; ++v)
      raw[i][v] = load_cache8<KIND>(place, c.dtype, min(h0 + i, c.hkv - 1), v != 0);
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    if (h0 + i >= c.hkv) break;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float x[8];
      cache8_values<KIND>(raw[i][v], c.dtype, x);
      if (page < 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
      }
      store8(v ? a.v_out : a.k_out, (static_cast<size_t>(r) * c.hkv + h0 + i) * HD + d, a.out_dtype,
             x, a.vec >> v & 1);
    }
  }
}

// Any head size: one warp per (token, KV head).
__global__ void __launch_bounds__(128) ragged_read_any_kernel(const __grid_constant__ RaggedReadArgs a) {
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const CacheView& c = a.cache;
  const int64_t r64 = warp / c.hkv;
  if (r64 >= a.rows.first[a.batch]) return;
  const int r = static_cast<int>(r64), h = static_cast<int>(warp - r64 * c.hkv);
  const int b = ragged_seq(a.rows, a.batch, r);
  bool ok;
  const int64_t row = cache_row(c, a.rows.seq[b], a.rows.start[b] + r - a.rows.first[b], h,
                                a.status, ok);
  const size_t o = static_cast<size_t>(warp) * c.hd;
  for (int d = threadIdx.x & 31; d < c.hd; d += 32) {
    store_elem(a.k_out, o + d, a.out_dtype, ok ? cache_value(c, false, row, d) : 0.f);
    store_elem(a.v_out, o + d, a.out_dtype, ok ? cache_value(c, true, row, d) : 0.f);
  }
}

cudaError_t launch_ragged_read(const RaggedReadArgs& a_in, cudaStream_t s) {
  RaggedReadArgs a = a_in;
  const int64_t tokens = a.rows.first[a.batch];
  if (tokens == 0) return cudaSuccess;
  a.vec = (reinterpret_cast<uintptr_t>(a.k_out) % 16 == 0 ? 1 : 0) |
          (reinterpret_cast<uintptr_t>(a.v_out) % 16 == 0 ? 2 : 0);
  const int hd = a.cache.hd, dt = a.cache.dtype;
  if (hd != 64 && hd != 128) {
    const int64_t threads = tokens * a.cache.hkv * 32;
    ragged_read_any_kernel<<<static_cast<unsigned>((threads + 127) / 128), 128, 0, s>>>(a);
    return cudaGetLastError();
  }
  const dim3 grid(static_cast<unsigned>((tokens * (hd / 8) + 255) / 256),
                  (a.cache.hkv + kAtOnce - 1) / kAtOnce);
  const auto k = hd == 64 ? dt == kQ4_0   ? ragged_read_kernel<64, kQ4_0>
                            : dt == kQ8_0 ? ragged_read_kernel<64, kQ8_0>
                                          : ragged_read_kernel<64, kF32>
                 : dt == kQ4_0 ? ragged_read_kernel<128, kQ4_0>
                 : dt == kQ8_0 ? ragged_read_kernel<128, kQ8_0>
                               : ragged_read_kernel<128, kF32>;
  k<<<grid, 256, 0, s>>>(a);
  return cudaGetLastError();
}

// ------------------------------------------------------ block selection --
namespace {

__device__ __forceinline__ size_t bounds_row(const CacheView& c, int page, int block, int kvh) {
  const int per = c.page / kTile;
  return ((static_cast<size_t>(page) * per + block % per) * c.hkv + kvh) * 2 * c.hd;
}

}  // namespace

// One CTA per (block, KV head): the least and largest key of each channel, rounded to f16 or
// bf16.  A channel that holds a NaN gets NaN bounds.  HD 64 or 128: HD / 8 lanes a position as in
// the append, the block's positions in rounds, joined over the groups through shared memory;
// HD 0: a thread a channel.
template <int HD, int KIND>
__global__ void __launch_bounds__(128) bounds_kernel(const __grid_constant__ BoundsArgs a) {
  const CacheView& c = a.cache;
  const int kvh = blockIdx.y;
  const int b = ragged_seq(a.blocks, a.batch, blockIdx.x);
  const int block = a.blocks.start[b] + static_cast<int>(blockIdx.x) - a.blocks.first[b];
  const int page = page_of(c, a.blocks.seq[b], block * kTile, a.status);
  if (page < 0) return;
  uint16_t* out = a.bounds + bounds_row(c, page, block, kvh);
  const bool half = c.dtype == kF16;
  auto write = [&](int d, float lo, float hi, bool nan) {
    if (nan) lo = hi = CUDART_NAN_F;
    out[d] = static_cast<uint16_t>(half ? pack2<false>(lo, lo) : pack2<true>(lo, lo));
    out[c.hd + d] = static_cast<uint16_t>(half ? pack2<false>(hi, hi) : pack2<true>(hi, hi));
  };
  if constexpr (HD != 0) {
    constexpr int kLanes = HD / 8, kGroups = 128 / kLanes;
    const int group = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 8;
    float lo[8], hi[8];
    uint32_t nan = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) lo[k] = CUDART_INF_F, hi[k] = -CUDART_INF_F;
#pragma unroll 4
    for (int i = group; i < kTile; i += kGroups) {
      float x[8];
      cache8_values<KIND>(
          load_cache8<KIND>(row_place<KIND>(c, page, block * kTile + i, d), c.dtype, kvh, false),
          c.dtype, x);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        nan |= (x[k] != x[k] ? 1u : 0u) << k;
        lo[k] = fminf(lo[k], x[k]);
        hi[k] = fmaxf(hi[k], x[k]);
      }
    }
    __shared__ float part[2][kGroups][HD];
    __shared__ uint32_t nans[kGroups][kLanes];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      part[0][group][d + k] = lo[k];
      part[1][group][d + k] = hi[k];
    }
    nans[group][d / 8] = nan;
    __syncthreads();
    for (int e = threadIdx.x; e < HD; e += 128) {
      float l = CUDART_INF_F, h = -CUDART_INF_F;
      uint32_t bad = 0;
      for (int g = 0; g < kGroups; ++g) {
        l = fminf(l, part[0][g][e]);
        h = fmaxf(h, part[1][g][e]);
        bad |= nans[g][e / 8];
      }
      write(e, l, h, bad >> (e % 8) & 1u);
    }
  } else {
    const int64_t row = (static_cast<int64_t>(page) * c.hkv + kvh) * c.page + block * kTile % c.page;
    for (int d = threadIdx.x; d < c.hd; d += 128) {
      float lo = CUDART_INF_F, hi = -CUDART_INF_F;
      bool nan = false;
      for (int i = 0; i < kTile; ++i) {
        const float x = cache_value(c, false, row + i, d);
        nan |= x != x;
        lo = fminf(lo, x);
        hi = fmaxf(hi, x);
      }
      write(d, lo, hi, nan);
    }
  }
}

namespace {

template <int HD>
auto bounds_form(int dtype) {
  return dtype == kQ4_0 ? bounds_kernel<HD, kQ4_0> : dtype == kQ8_0 ? bounds_kernel<HD, kQ8_0>
                                                                    : bounds_kernel<HD, kF32>;
}

}  // namespace

cudaError_t launch_bounds(const BoundsArgs& a, cudaStream_t s) {
  const int n = a.blocks.first[a.batch];
  if (n == 0) return cudaSuccess;
  const auto k = a.cache.hd == 128  ? bounds_form<128>(a.cache.dtype)
                 : a.cache.hd == 64 ? bounds_form<64>(a.cache.dtype)
                                    : bounds_kernel<0, kF32>;
  k<<<dim3(n, a.cache.hkv), 128, 0, s>>>(a);
  return cudaGetLastError();
}

namespace {

constexpr int kChooseThreads = 256;
constexpr int kBins = 2048;

constexpr int kMaxChunk = 256;  // blocks that a CTA scores at most

// Eight consecutive values of a bounds row.
__device__ __forceinline__ void bounds_values(const uint4& w, bool half, float (&x)[8]) {
  const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = half ? __half22float2(*reinterpret_cast<const __half2*>(&in[k]))
                          : make_float2(__uint_as_float(in[k] << 16),
                                        __uint_as_float(in[k] & 0xffff0000u));
    x[2 * k] = f.x, x[2 * k + 1] = f.y;
  }
}

// Adds query value x to the sums of a channel's positive and negative parts.
__device__ __forceinline__ void add_parts(float x, double& up, double& down) {
  if (x > 0.f) up += x;
  else down += x;  // a NaN lands here
}

// Channels d0, d0 + step .. below end of one block's score by its definition, head for head, a
// NaN passed on.  For the blocks whose score by parts is a NaN: there 0 times an infinite bound
// may stand for queries that the group does not have.
__device__ __noinline__ double score_by_heads(const void* q, size_t q0, int in_dtype, int group,
                                              int hd, const uint16_t* bounds, int bound_dtype,
                                              int d0, int step, int end) {
  double s = 0.0;
  for (int d = d0; d < end; d += step) {
    const double lo = load_elem(bounds, d, bound_dtype), hi = load_elem(bounds, hd + d, bound_dtype);
    for (int h = 0; h < group; ++h) {
      const double x = load_elem(q, q0 + static_cast<size_t>(h) * hd + d, in_dtype);
      const double a = x * lo, b = x * hi;
      s += a != a ? a : b != b ? b : fmax(a, b);
    }
  }
  return s;
}

// The least and the largest over the block's threads.
__device__ __forceinline__ void block_range(double& least, double& most, double2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    least = fmin(least, __shfl_xor_sync(0xffffffffu, least, o));
    most = fmax(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_double2(least, most);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kChooseThreads / 32; ++i) {
    least = fmin(least, red[i].x);
    most = fmax(most, red[i].y);
  }
}

}  // namespace

// Scores and choice in one launch.  The CTAs of a (token, KV head) score a.chunk blocks each;
// the last to arrive chooses.
//
// Scores: the group's queries enter by the sums of their positive and of their negative parts,
// because sum_h max(q_h lo, q_h hi) = (sum_h max(q_h, 0)) hi + (sum_h min(q_h, 0)) lo while
// lo <= hi are finite: two products a channel whatever the group.  In f64, so that only equal
// blocks tie.  An infinite bound times a sum that is 0 for want of queries gives a NaN, and any
// NaN sends the block to score_by_heads.
// HD / 8 lanes a block (HD 64 or 128), else (HD 0) a warp.  A block whose table entry is
// outside the pool raises the status and scores the least, so that every score is written and
// none is a NaN: the ranks below are then those of distinct places.
//
// Choice: a histogram over the range of the scores puts the border into one of kBins bins;
// those above it are in, and the few in it are ranked among themselves by (score, block).
//
// Bound by latencies: the queries, the pages, the bounds, the count, then the passes of the last
// CTA (about 5 us): 12 us for 8 KV heads of 512 blocks, 18 us for 64 of up to 781 (31,000
// blocks, 16 MB of bounds).  A rank of every score by comparison with all took 100 us there.
template <int HD>
__global__ void __launch_bounds__(kChooseThreads)
    choose_kernel(const __grid_constant__ SelectArgs a) {
  const CacheView& c = a.cache;
  const int kvh = blockIdx.y, job = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = job / a.new_len, qpos = a.seqs.start[b] + job % a.new_len;
  const int count = qpos / kTile + 1;
  const size_t pair = static_cast<size_t>(job) * c.hkv + kvh;
  int32_t* sel = a.sel + pair * a.take;
  griddep_wait();
  griddep_launch_dependents();
  if (count <= a.take) {  // all of them
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i < a.take; i += kChooseThreads) sel[i] = i < count ? i : -1;
    return;
  }
  const int lo_block = a.first, hi_block = count - a.last;  // the candidates
  const int chunks = (hi_block + a.chunk - 1) / a.chunk;
  if (static_cast<int>(blockIdx.x) >= chunks) return;
  const int free = a.take - a.first - a.last;
  double* score = a.score + pair * a.max_blocks;

  // ---------------------------------------------------------------- scores --
  if (free > 0) {
    const int32_t* table = c.block_table + static_cast<size_t>(a.seqs.seq[b]) * c.pages_per_seq;
    const size_t q0 = (static_cast<size_t>(job) * a.hq + kvh * a.group) * c.hd;
    const bool half = c.dtype == kF16;
    auto bounds_of = [&](int block) -> const uint16_t* {
      const int page = table[block * kTile / c.page];
      if (page < 0 || page >= c.num_pages) {
        atomicOr(a.status, kStatusBadPage);
        return nullptr;
      }
      return a.bounds + bounds_row(c, page, block, kvh);
    };
    const int block0 = blockIdx.x * a.chunk, end = min(block0 + a.chunk, hi_block);
    if constexpr (HD != 0) {
      constexpr int kLanes = HD / 8;  // of a block: lane `sub` has dims 8 sub .. + 7
      const int sub = lane & (kLanes - 1);
      double up[8], down[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) up[k] = down[k] = 0.0;
      constexpr int kHeads = 4;  // loaded at once
      for (int h0 = 0; h0 < a.group; h0 += kHeads) {
        Raw8 raw[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
          raw[h] = load_raw8(a.q, q0 + static_cast<size_t>(min(h0 + h, a.group - 1)) * HD + 8 * sub,
                             a.in_dtype, a.q_vec != 0);
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          float x[8];
          floats_of(raw[h], a.in_dtype, x);
          if (h0 + h < a.group) {
#pragma unroll
            for (int k = 0; k < 8; ++k) add_parts(x[k], up[k], down[k]);
          }
        }
      }
      // The blocks of all rounds are looked up at once, one by each lane of a group, and the
      // next round's bounds are under way while one is summed.
      constexpr int kRound = kChooseThreads / kLanes;
      static_assert(kMaxChunk <= kLanes * kRound, "a lane a round");
      const int base = block0 + 32 / kLanes * warp + lane / kLanes;
      const uint16_t* mine = nullptr;
      if (base + sub * kRound < end && base + sub * kRound >= lo_block)
        mine = bounds_of(base + sub * kRound);
      struct Bounds {
        uint4 lo, hi;
        const uint16_t* p;
      };
      auto fetch = [&](int round) {
        Bounds x;
        x.p = reinterpret_cast<const uint16_t*>(__shfl_sync(
            0xffffffffu, reinterpret_cast<unsigned long long>(mine), (lane & ~(kLanes - 1)) + round));
        if (x.p) {
          x.lo = *reinterpret_cast<const uint4*>(x.p + 8 * sub);
          x.hi = *reinterpret_cast<const uint4*>(x.p + HD + 8 * sub);
        }
        return x;
      };
      const int rounds = (end - block0 + kRound - 1) / kRound;
      Bounds next = fetch(0);
      for (int round = 0; round < rounds; ++round) {
        const Bounds x = next;
        if (round + 1 < rounds) next = fetch(round + 1);
        double s[2] = {};
        if (x.p) {
          float lo[8], hi[8];
          bounds_values(x.lo, half, lo);
          bounds_values(x.hi, half, hi);
#pragma unroll
          for (int k = 0; k < 8; ++k) s[k & 1] += up[k] * hi[k] + down[k] * lo[k];
        }
        double t = s[0] + s[1];
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (__any_sync(0xffffffffu, t != t)) {
          double e = 0.0;
          if (t != t)
            e = score_by_heads(a.q, q0, a.in_dtype, a.group, HD, x.p, half ? kF16 : kBF16, 8 * sub,
                               1, 8 * sub + 8);
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) e += __shfl_xor_sync(0xffffffffu, e, o);
          if (t != t) t = e == e ? e : CUDART_INF;  // a NaN counts as the largest score
        }
        if (!x.p) t = -CUDART_INF;  // on no page: flagged, and chosen last
        const int block = base + round * kRound;
        if (sub == 0 && block >= lo_block && block < end) score[block] = t;
      }
    } else {
      const int bt = half ? kF16 : kBF16;
      for (int block = max(block0, lo_block) + warp; block < end; block += kChooseThreads / 32) {
        const uint16_t* p = bounds_of(block);
        double s = 0.0;
        for (int d = lane; p && d < c.hd; d += 32) {
          double up = 0.0, down = 0.0;
          for (int h = 0; h < a.group; ++h)
            add_parts(load_elem(a.q, q0 + static_cast<size_t>(h) * c.hd + d, a.in_dtype), up, down);
          s += up * load_elem(p, c.hd + d, bt) + down * load_elem(p, d, bt);
        }
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (s != s) {  // (every lane alike)
          s = score_by_heads(a.q, q0, a.in_dtype, a.group, c.hd, p, bt, lane, 32, c.hd);
          for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          if (s != s) s = CUDART_INF;
        }
        if (lane == 0) score[block] = p ? s : -CUDART_INF;
      }
    }
  }
  // The barrier orders the CTA's scores before thread 0's count, whose release makes them
  // visible; the last CTA's acquire sees the others'.
  __shared__ int flag[4];  // last one to arrive; the border's bin, how many lie above it; border list
  __syncthreads();
  if (threadIdx.x == 0)
    flag[0] = chunks == 1 || atom_add_acq_rel_gpu(&a.counters[pair], 1) == chunks - 1;
  __syncthreads();
  if (!flag[0]) return;
  if (threadIdx.x == 0) a.counters[pair] = 0;

  // ---------------------------------------------------------------- choice --
  extern __shared__ double dyn[];
  const bool fits = a.max_blocks <= a.smem_blocks;  // the scores, copied for the passes over them
  uint32_t* in = reinterpret_cast<uint32_t*>(dyn + (fits ? a.max_blocks : 0));  // a bit per block
  __shared__ int hist[kBins];
  __shared__ double2 red[kChooseThreads / 32];
  __shared__ int scan[kChooseThreads / 32];
  constexpr int kList = 512;
  __shared__ int list[kList];
  const int words = (count + 31) / 32;
  for (int i = threadIdx.x; i < kBins; i += kChooseThreads) hist[i] = 0;
  for (int i = threadIdx.x; i < words; i += kChooseThreads) {
    uint32_t w = 0;
    for (int k = 0; k < 32; ++k) {
      const int j = 32 * i + k;
      w |= (j < lo_block || (j >= hi_block && j < count) ? 1u : 0u) << k;
    }
    in[i] = w;
  }
  if (threadIdx.x == 0) flag[3] = 0;
  if (free > 0) {
    double least = CUDART_INF, most = -CUDART_INF;
#pragma unroll 4
    for (int j = lo_block + threadIdx.x; j < hi_block; j += kChooseThreads) {
      const double s = __ldcg(score + j);
      if (fits) dyn[j] = s;
      if (fabs(s) < CUDART_INF) {
        least = fmin(least, s);
        most = fmax(most, s);
      }
    }
    block_range(least, most, red);
    const double scale = most > least ? (kBins - 3) / (most - least) : 0.0;
    // (rounded differences and products keep the order; infinities have bins of their own)
    auto bin = [&](double s) {
      if (!(fabs(s) < CUDART_INF)) return s > 0.0 ? kBins - 1 : 0;
      return 1 + min(kBins - 3, static_cast<int>((s - least) * scale));
    };
    auto at = [&](int j) { return fits ? dyn[j] : __ldcg(score + j); };
    for (int j = lo_block + threadIdx.x; j < hi_block; j += kChooseThreads) atomicAdd(&hist[bin(at(j))], 1);
    __syncthreads();
    // Thread t's bins, from the top: kBins - 1 - 8 t .. ; how many scores lie above them.
    constexpr int kEach = kBins / kChooseThreads;
    int mine = 0;
    for (int k = 0; k < kEach; ++k) mine += hist[kBins - 1 - kEach * threadIdx.x - k];
    int above = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, above, o);
      if (lane >= o) above += up;
    }
    if (lane == 31) scan[warp] = above;
    __syncthreads();
    above -= mine;
    for (int w = 0; w < warp; ++w) above += scan[w];
    if (above < free && above + mine >= free) {
      int k = kBins - 1 - kEach * threadIdx.x;
      while (above + hist[k] < free) above += hist[k--];
      flag[1] = k;
      flag[2] = above;
    }
    __syncthreads();
    const int border = flag[1], need = free - flag[2];
    for (int j = lo_block + threadIdx.x; j < hi_block; j += kChooseThreads) {
      const int k = bin(at(j));
      if (k > border) {
        atomicOr(&in[j / 32], 1u << (j % 32));
      } else if (k == border) {
        const int n = atomicAdd(&flag[3], 1);
        if (n < kList) list[n] = j;
      }
    }
    __syncthreads();
    const int members = flag[3];
    if (members <= kList) {
      for (int i = threadIdx.x; i < members; i += kChooseThreads) {
        const int j = list[i];
        const double s = at(j);
        int rank = 0;
        for (int k = 0; k < members; ++k) {
          const double o = at(list[k]);
          rank += o > s || (o == s && list[k] < j);
        }
        if (rank < need) atomicOr(&in[j / 32], 1u << (j % 32));
      }
    } else {  // many equal scores
      for (int j = lo_block + threadIdx.x; j < hi_block; j += kChooseThreads) {
        const double s = at(j);
        if (bin(s) != border) continue;
        int rank = 0;
        for (int k = lo_block; k < hi_block && rank < need; ++k) {
          const double o = at(k);
          rank += bin(o) == border && (o > s || (o == s && k < j));
        }
        if (rank < need) atomicOr(&in[j / 32], 1u << (j % 32));
      }
    }
  }
  __syncthreads();
  if (warp != 0) return;
  for (int w0 = 0, done = 0; w0 < words; w0 += 32) {  // a word of the bits a lane
    uint32_t w = w0 + lane < words ? in[w0 + lane] : 0;
    const int n = __popc(w);
    int before = n;
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    for (int i = done + before - n; w; w &= w - 1, ++i)
      if (i < a.take) sel[i] = 32 * (w0 + lane) + __ffs(w) - 1;
    done += __shfl_sync(0xffffffffu, before, 31);
  }
}

cudaError_t launch_select(const SelectArgs& a_in, cudaStream_t s) {
  SelectArgs a = a_in;
  const int jobs = a.batch * a.new_len;
  // 48 KB of dynamic shared memory need no opt-in: the bits of every block, and the scores
  // while they fit beside them.
  const size_t bits = static_cast<size_t>((a.max_blocks + 31) / 32) * sizeof(uint32_t);
  constexpr size_t kLimit = 32 * 1024;
  a.smem_blocks = bits < kLimit ? static_cast<int32_t>((kLimit - bits) / sizeof(double)) : 0;
  const size_t smem = bits + (a.max_blocks <= a.smem_blocks ? a.max_blocks * sizeof(double) : 0);
  // Blocks of a CTA: 32 while the CTAs are few, more where they would come in several waves (a
  // CTA begins with the queries, whatever it scores).
  const int64_t pairs = static_cast<int64_t>(jobs) * a.cache.hkv;
  a.chunk = 32;
  while (a.chunk < kMaxChunk && pairs * ((a.max_blocks + a.chunk - 1) / a.chunk) > 4LL * a.num_sms) a.chunk *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.max_blocks + a.chunk - 1) / a.chunk, a.cache.hkv, jobs);
  cfg.blockDim = dim3(kChooseThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const auto k = a.cache.hd == 128  ? choose_kernel<128>
                 : a.cache.hd == 64 ? choose_kernel<64>
                                    : choose_kernel<0>;
  return cudaLaunchKernelEx(&cfg, k, a);
}

}  // namespace ql
