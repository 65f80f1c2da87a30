// ql_linear.cu -- the layers of a decode step on 4-bit weights
// (qllama_model.h): RMSNorm with the residual's addition and an optional Q8_0
// output, the 4-bit weight matrices, and products of a few rows with them.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>

#include "../../include/qllama_model.h"
#include "ql_device.cuh"
#include "ql_internal.h"

namespace {

#define QLN_CUDA(call, what)                                                                   \
  do {                                                                                         \
    cudaError_t e_ = (call);                                                                   \
    if (e_ != cudaSuccess) {                                                                   \
      cudaGetLastError(); /* a refused allocation is not the next launch's error */            \
      return ql_fail(e_ == cudaErrorMemoryAllocation ? QL_ERR_OOM : QL_ERR_CUDA, "%s: %s",    \
                     what, cudaGetErrorString(e_));                                            \
    }                                                                                          \
  } while (0)

bool float_type(int dt) { return dt == QL_F32 || dt == QL_F16 || dt == QL_BF16; }
size_t type_bytes(int dt) { return dt == QL_F32 ? 4 : dt == QL_Q8_0 ? 1 : 2; }
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// ------------------------------------------------------------------ RMSNorm --

struct NormArgs {
  const void* x;
  const void* residual;
  const void* weight;
  void* sum_out;
  void* out;
  __half* out_scale;
  int64_t x_stride, residual_stride;
  int rows, hidden, in_dtype, weight_dtype, out_dtype;
  float eps, inv_hidden;
};

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the CTA (every thread gets it, in the same order of additions).
template <typename T>
__device__ __forceinline__ T block_sum(T v, T* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int l = threadIdx.x & 31;
  return warp_sum(l < static_cast<int>(blockDim.x >> 5) ? red[l] : T(0));
}

// Whether an f32 sum of squares can be used as it is: neither overflowed (or
// NaN) nor so small that squares below f32's normal range were a part of it.
__device__ __forceinline__ bool plain_square_sum(float ss) {
  return ss >= 0x1p-80f && ss < 0x1p126f;
}

// round(v), ties away from zero, for |v| < 2^22: the largest f32 below 0.5 is
// added away from zero and the sum is cut.  (With 0.5 itself, values just below
// a tie would be carried over it; v = 0.5 still reaches 1, since the sum rounds.)
__device__ __forceinline__ int round_away(float v) {
  return __float2int_rz(v + copysignf(0x1.fffffep-2f, v));
}

// Magnitudes as integers: they order like the values, and a NaN or an infinity
// is above every finite one, so that one maximum carries both.
__device__ __forceinline__ uint32_t magnitude(float y) { return __float_as_uint(y) & 0x7fffffffu; }

__device__ __forceinline__ float rcp_fast(float v) {  // within 1 ulp
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// Q8_0 scale d of a block whose largest magnitude is `most`, and inv = 1 / d.  The two
// divisions of the rule are a product with 1/127 and an approximate reciprocal, each
// within an ulp (they were a tenth of the instructions).  A value y / d, 127 at most, is
// then off by 127 * 3 * 2^-23 or less: next to a tie it may go to the other side.  `limit` is where values are
// cut: finite only if the scale saturates, 0 for a block with a NaN or an infinity.
__device__ __forceinline__ __half q8_scale(uint32_t most, float& inv, float& limit) {
  float d = __uint_as_float(most) * (1.0f / 127.0f);
  limit = INFINITY;
  if (most >= 0x7f800000u) {
    limit = inv = 0.f;
    return __ushort_as_half(0x7fff);
  }
  if (d > 65504.0f) {
    d = 65504.0f;
    limit = 127.0f * 65504.0f;
  }
  inv = d > 1e-30f ? rcp_fast(d) : 0.f;  // (as f16 it is 0 long before)
  return __float2half_rn(d);
}

__device__ __forceinline__ float q8_cut(float y, float limit) {
  return limit == 0.f ? 0.f : fminf(fmaxf(y, -limit), limit);
}

// One CTA per row, element by element, reading the row twice: what the kernel
// below cannot take (more columns than it holds, tensors that do not start on
// 16 bytes, strides that break the groups of eight).
constexpr int kNormThreads = 256;
__global__ void __launch_bounds__(kNormThreads) rms_norm_loop_kernel(const NormArgs a) {
  __shared__ float red[32];
  __shared__ double red_d[32];
  const size_t row = blockIdx.x;
  const size_t xo = row * static_cast<size_t>(a.x_stride);
  const size_t ro = row * static_cast<size_t>(a.residual_stride);
  const size_t oo = row * static_cast<size_t>(a.hidden);
  ql::griddep_wait();
  ql::griddep_launch_dependents();
  auto value = [&](int i) {
    float s = ql::load_elem(a.x, xo + i, a.in_dtype);
    if (a.residual) s += ql::load_elem(a.residual, ro + i, a.in_dtype);
    return s;
  };
  float ss = 0.f;
  for (int i = threadIdx.x; i < a.hidden; i += kNormThreads) {
    const float s = value(i);
    ss += s * s;
  }
  ss = block_sum(ss, red);
  const bool plain = plain_square_sum(ss);
  float inv = rsqrtf(fmaf(ss, a.inv_hidden, a.eps));  // within 2 ulp
  double inv_d = 0.0;
  if (!plain) {
    double sd = 0.0;
    for (int i = threadIdx.x; i < a.hidden; i += kNormThreads) {
      const double s = value(i);
      sd += s * s;
    }
    inv_d = 1.0 / sqrt(block_sum(sd, red_d) / a.hidden + static_cast<double>(a.eps));
  }
  const int n = (a.hidden + kNormThreads - 1) / kNormThreads * kNormThreads;
  for (int i = threadIdx.x; i < n; i += kNormThreads) {  // whole warps: the shuffles below
    float y = 0.f;
    if (i < a.hidden) {
      const float s = value(i);
      const float w = ql::load_elem(a.weight, i, a.weight_dtype);
      if (a.sum_out) ql::store_elem(a.sum_out, oo + i, a.in_dtype, s);
      y = plain ? s * inv * w : static_cast<float>(s * inv_d * w);
      if (a.out_dtype != ql::kQ8_0) ql::store_elem(a.out, oo + i, a.out_dtype, y);
    }
    if (a.out_dtype == ql::kQ8_0) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, magnitude(y));
      if (i < a.hidden) {
        float id, limit;
        const __half d = q8_scale(m, id, limit);
        if (limit != INFINITY) y = q8_cut(y, limit);
        static_cast<int8_t*>(a.out)[oo + i] = static_cast<int8_t>(round_away(y * id));
        if (i % 32 == 0) a.out_scale[(oo + i) / 32] = d;
      }
    }
  }
}

// Eight consecutive elements: 16 bytes, or 32 for f32.
template <int DT>
struct Raw8 {
  static constexpr int kWords = DT == ql::kF32 ? 8 : 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* base, size_t i) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(base) +
                                                    i * (DT == ql::kF32 ? 4 : 2));
#pragma unroll
    for (int j = 0; j < kWords / 4; ++j) {
      const uint4 v = p[j];
      w[4 * j] = v.x;
      w[4 * j + 1] = v.y;
      w[4 * j + 2] = v.z;
      w[4 * j + 3] = v.w;
    }
  }
  // elements [lo, hi) of the eight one by one, zeros for the others
  __device__ __forceinline__ void load_part(const void* base, size_t i, int lo, int hi) {
#pragma unroll
    for (int j = 0; j < kWords; ++j) w[j] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e < lo || e >= hi) continue;
      if constexpr (DT == ql::kF32)
        w[e] = static_cast<const uint32_t*>(base)[i + e];
      else
        w[e / 2] |= static_cast<uint32_t>(static_cast<const uint16_t*>(base)[i + e])
                    << (16 * (e & 1));
    }
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (DT == ql::kF32) {
        x[e] = __uint_as_float(w[e]);
      } else {
        const uint16_t h = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
        if constexpr (DT == ql::kF16) x[e] = __half2float(__ushort_as_half(h));
        else x[e] = __uint_as_float(static_cast<uint32_t>(h) << 16);
      }
    }
  }
};

__device__ __forceinline__ void store_part(void* base, size_t i, int dt, const float (&x)[8],
                                           int lo, int hi) {
  if (lo == 0 && hi == 8) return ql::store8(base, i, dt, x, true);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e >= lo && e < hi) ql::store_elem(base, i + e, dt, x[e]);
}

// One CTA per row; a thread holds NV groups of eight columns in registers, so
// that x and the residual are read once, all loads of a row in flight together,
// and the row's sum and result are written once.  Bound by those bytes for many
// rows and by one round trip to memory plus the reduction for a few; launch_norm
// says how NV is chosen.
// LEAD: the row length is no multiple of eight, so a row starts `lead` elements
// into an aligned group of eight.  Groups keep that alignment -- it is the same
// in every contiguous tensor, whatever its type -- and only the row's first and
// last go element by element (2000 rows of 4101 bf16 columns 19.2 us, 52.8 us
// with element-wise loads throughout).
// WARP: a warp per row, kNormRows rows to a CTA, for many short rows (8000 x 128 bf16 with
// a residual 8.6 us with a CTA for each, 2.9 us so; 8000 x 512 9.0 us and 6.3 us; 8000 x
// 1000 12.5 us and 15.4 us).
constexpr int kNormMax = 16384;  // 512 threads x 32 columns
constexpr int kNormRows = 8;
template <int DT, int WT, int NV, bool LEAD, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kNormRows : NV == 1 ? 1024 : 512,
                                  !WARP && NV > 1 ? 2 : 1)
    rms_norm_kernel(const NormArgs a) {
  __shared__ float red[32];
  __shared__ double red_d[32];
  const size_t row = WARP ? blockIdx.x * static_cast<size_t>(kNormRows) + threadIdx.x / 32
                          : blockIdx.x;
  const int thread = WARP ? threadIdx.x % 32 : threadIdx.x;
  const int threads = WARP ? 32 : blockDim.x;
  const size_t oo = row * static_cast<size_t>(a.hidden);
  const int lead = LEAD ? static_cast<int>(oo % 8) : 0;
  ql::griddep_wait();
  ql::griddep_launch_dependents();
  if (WARP && row >= static_cast<size_t>(a.rows)) return;
  // where x and the residual fill the registers, the weight is left for later
  constexpr bool kEarly = NV * (DT == ql::kF32 ? 2 : 1) < 4;
  Raw8<DT> xr[NV], rr[NV];
  Raw8<WT> wr[NV];
  auto column = [&](int j) { return 8 * (thread + j * threads) - lead; };
  auto read = [&](auto& r, const void* base, size_t at, int c, bool whole) {
    if (!LEAD || whole) r.load(base, at + c);
    else r.load_part(base, at + c, c < 0 ? -c : 0, min(8, a.hidden - c));
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = column(j);
    if (c < a.hidden) {
      const bool whole = c >= 0 && c + 8 <= a.hidden;
      read(xr[j], a.x, row * static_cast<size_t>(a.x_stride), c, whole);
      if (a.residual) read(rr[j], a.residual, row * static_cast<size_t>(a.residual_stride), c, whole);
    }
  }
  if constexpr (kEarly) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (column(j) < a.hidden) read(wr[j], a.weight, 0, column(j), lead == 0 && column(j) + 8 <= a.hidden);
  }
  float s[NV][8];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = column(j);
    if (c < a.hidden) {
      xr[j].get(s[j]);
      if (a.residual) {
        float r[8];
        rr[j].get(r);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j][e] += r[e];
        if (a.sum_out)
          store_part(a.sum_out, oo + c, DT, s[j], LEAD && c < 0 ? -c : 0,
                     LEAD ? min(8, a.hidden - c) : 8);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += s[j][e] * s[j][e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[j][e] = 0.f;
    }
  }
  ss = WARP ? warp_sum(ss) : block_sum(ss, red);
  float inv = rsqrtf(fmaf(ss, a.inv_hidden, a.eps));  // within 2 ulp
  if (!plain_square_sum(ss)) {
    // the same for every thread: 64 bits, and s becomes s * inv here
    double sd = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sd += static_cast<double>(s[j][e]) * s[j][e];
    sd = WARP ? warp_sum(sd) : block_sum(sd, red_d);
    const double id = 1.0 / sqrt(sd / a.hidden + static_cast<double>(a.eps));
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[j][e] = static_cast<float>(s[j][e] * id);
    inv = 1.f;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = column(j);
    const bool in = c < a.hidden;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = 0.f;
    if (in) {
      float w[8];
      if constexpr (!kEarly) read(wr[j], a.weight, 0, c, lead == 0 && c + 8 <= a.hidden);
      wr[j].get(w);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = s[j][e] * inv * w[e];
    }
    if (LEAD || a.out_dtype != ql::kQ8_0) {
      if (in)
        store_part(a.out, oo + c, a.out_dtype, y, LEAD && c < 0 ? -c : 0,
                   LEAD ? min(8, a.hidden - c) : 8);
      continue;
    }
    // a block of 32 columns is four neighbouring lanes' (hidden % 32 == 0:
    // all four inside the row, or none)
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, magnitude(y[e]));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    float id, limit;
    const __half d = q8_scale(m, id, limit);
    if (limit != INFINITY) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = q8_cut(y[e], limit);
    }
    uint32_t q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = static_cast<uint32_t>(round_away(y[e] * id));
    if (in) {
      uint2 w;
      w.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
      w.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
      *reinterpret_cast<uint2*>(static_cast<int8_t*>(a.out) + oo + c) = w;
      if ((threadIdx.x & 3) == 0) a.out_scale[(oo + c) / 32] = d;
    }
  }
}

// A launch that may begin while the kernel before it in the stream drains
// (every kernel here waits for that kernel's end before it touches a tensor; only a
// product's weights are read ahead).
template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                       A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// NV: a few rows go over as many threads as they have groups (one round trip,
// the shortest reduction); with two rows or more for every SM, twice as many
// columns a thread (fewer threads wait in a reduction: 4099 x 4096 bf16 22.1 us, 30.7 us
// with one group a thread).
cudaError_t launch_norm(const NormArgs& a, int num_sms, cudaStream_t s) {
  auto fits = [](const void* p, int dt, int64_t stride) {
    const size_t to = dt == QL_Q8_0 ? 8 : 16;
    return aligned(p, to) && (stride * type_bytes(dt)) % to == 0;
  };
  const bool bases = aligned(a.x, 16) && aligned(a.residual, 16) && aligned(a.sum_out, 16) &&
                     aligned(a.weight, 16) && aligned(a.out, a.out_dtype == QL_Q8_0 ? 8 : 16);
  const bool even = a.hidden % 8 == 0 && fits(a.x, a.in_dtype, a.x_stride) &&
                    (!a.residual || fits(a.residual, a.in_dtype, a.residual_stride));
  const bool lead = !even && a.hidden % 8 != 0 && a.x_stride == a.hidden &&
                    (!a.residual || a.residual_stride == a.hidden);
  if (!bases || !(even || lead) || a.hidden > kNormMax - 8)
    return launch_pdl(rms_norm_loop_kernel, dim3(a.rows), dim3(kNormThreads), 0, s, a);
  const int groups = (a.hidden + 7) / 8 + lead;
  const bool warp = groups <= 64 && a.rows >= 4 * num_sms;
  int nv = warp ? (groups <= 32 ? 1 : 2) : groups <= 1024 ? 1 : 4;
  if (nv == 1 && a.rows >= 2 * num_sms && groups >= 256) nv = 2;
  const dim3 block(warp ? 32 * kNormRows : ((groups + nv - 1) / nv + 31) / 32 * 32);
  const dim3 grid(warp ? (a.rows - 1) / kNormRows + 1 : a.rows);
  auto go = [&](auto dt, auto wt, auto ld) {
    constexpr int DT = decltype(dt)::value, WT = decltype(wt)::value;
    constexpr bool LEAD = decltype(ld)::value;
    auto* const kernel = warp ? (nv == 1 ? rms_norm_kernel<DT, WT, 1, LEAD, true>
                                         : rms_norm_kernel<DT, WT, 2, LEAD, true>)
                         : nv == 1 ? rms_norm_kernel<DT, WT, 1, LEAD, false>
                         : nv == 2 ? rms_norm_kernel<DT, WT, 2, LEAD, false>
                                   : rms_norm_kernel<DT, WT, 4, LEAD, false>;
    return launch_pdl(kernel, grid, block, 0, s, a);
  };
  auto by_lead = [&](auto dt, auto wt) {
    return lead ? go(dt, wt, std::true_type()) : go(dt, wt, std::false_type());
  };
  auto by_weight = [&](auto dt) {
    switch (a.weight_dtype) {
      case QL_F32: return by_lead(dt, std::integral_constant<int, ql::kF32>());
      case QL_F16: return by_lead(dt, std::integral_constant<int, ql::kF16>());
      default: return by_lead(dt, std::integral_constant<int, ql::kBF16>());
    }
  };
  switch (a.in_dtype) {
    case QL_F32: return by_weight(std::integral_constant<int, ql::kF32>());
    case QL_F16: return by_weight(std::integral_constant<int, ql::kF16>());
    default: return by_weight(std::integral_constant<int, ql::kBF16>());
  }
}

}  // namespace

// ------------------------------------------------------------- 4-bit weights --
// Device order.  Tiles of 16 rows x 64 columns, row tiles outermost, so that a
// row tile is one contiguous stream along the columns.  Tile (tile, chunk) is
// 32 lanes x 4 words: lane = 4 g + t, word i = 2 j + h holds row
// 16 tile + g + 8 h, columns 64 chunk + 32 j + 8 t .. + 7 -- the lane that needs
// them in the A fragment of an m16n8k16 / m16n8k32 product (any order of the
// columns inside a fragment serves, if x follows it).  A word holds the eight
// values (code - 8) as two's-complement nibbles in the order of nibble_of.  Scales:
// f16, one for each row and group of 32 columns (64 bytes a tile, [g][j][h]), of
// 64 (32 bytes a tile, [g][h]) or of 128 (32 bytes for two tiles along the columns);
// the four lanes of a quad read the same.
struct ql_q4 {
  ql_ctx* ctx = nullptr;
  int n = 0, k = 0, group = 0;
  int tiles = 0, chunks = 0;
  uint32_t* codes = nullptr;   // [tiles][chunks][32][4]
  __half* scales = nullptr;    // [tiles][chunks][8][2][2], [tiles][chunks or chunks/2][8][2]
};

namespace {

// Nibble that holds element e of a word's eight: (0,4) (2,6) (1,5) (3,7) are
// the pairs that a mask of 0x000f000f leaves after shifts of 0, 8, 4 and 12.
__host__ __device__ constexpr int nibble_of(int e) {
  return (e & 1) * 4 + (e >> 1 & 1) * 2 + (e >> 2);
}

struct Q4View {
  uint32_t* codes;
  __half* scales;
  int n, k, group, tiles, chunks;
};

Q4View view_of(const ql_q4* w) {
  return {w->codes, w->scales, w->n, w->k, w->group, w->tiles, w->chunks};
}

size_t q4_words(const ql_q4* w) { return static_cast<size_t>(w->tiles) * w->chunks * 128; }
size_t q4_scales(const ql_q4* w) {
  const size_t tiles = static_cast<size_t>(w->tiles) * w->chunks;
  return w->group == 32 ? tiles * 32 : w->group == 64 ? tiles * 16 : tiles * 8;
}

// Place of the scale of row g + 8 h and 32 columns j of tile (tile, chunk).
__host__ __device__ __forceinline__ size_t scale_at(int group, int chunks, size_t tile, int chunk,
                                                    int g, int j, int h) {
  if (group == 32) return ((tile * chunks + chunk) * 8 + g) * 4 + 2 * j + h;
  if (group == 64) return ((tile * chunks + chunk) * 8 + g) * 2 + h;
  return ((tile * (chunks / 2) + chunk / 2) * 8 + g) * 2 + h;
}

// Row and first column of word i of lane `lane` of tile (tile, chunk).
__device__ __forceinline__ void word_place(size_t tile, int chunk, int lane, int i, int& row,
                                           int& col) {
  row = static_cast<int>(tile) * 16 + (lane >> 2) + 8 * (i & 1);
  col = chunk * 64 + 32 * (i >> 1) + 8 * (lane & 3);
}

enum PackFrom : int { kPackCodes = 0, kPackBlocks = 1, kPackDense = 2 };

struct PackArgs {
  Q4View w;
  const uint8_t* bytes;  // codes or blocks
  const uint16_t* scales;
  const void* dense;     // element (row, col) at row * row_stride + col * col_stride
  int64_t row_stride, col_stride;
  int dtype;
};

// One thread per word of the device order.
template <int FROM>
__global__ void __launch_bounds__(256) q4_pack_kernel(const PackArgs a) {
  const size_t id = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  const size_t per_tile = static_cast<size_t>(a.w.chunks) * 128;
  if (id >= per_tile * a.w.tiles) return;
  const size_t tile = id / per_tile;
  const int rest = static_cast<int>(id % per_tile);
  const int chunk = rest >> 7, lane = rest >> 2 & 31, i = rest & 3;
  int row, col;
  word_place(tile, chunk, lane, i, row, col);
  uint32_t word = 0;
  uint16_t scale = 0;
  if (row < a.w.n && col < a.w.k) {
    if constexpr (FROM == kPackCodes) {
      const uint8_t* p = a.bytes + (static_cast<size_t>(row) * a.w.k + col) / 2;
      for (int e = 0; e < 8; ++e) {
        const uint32_t c = (p[e >> 1] >> (4 * (e & 1))) & 15u;
        word |= (c ^ 8u) << (4 * nibble_of(e));
      }
      scale = a.scales[static_cast<size_t>(row) * (a.w.k / a.w.group) + col / a.w.group];
    } else if constexpr (FROM == kPackBlocks) {
      const uint8_t* b = a.bytes + (static_cast<size_t>(row) * (a.w.k / 32) + col / 32) * 18;
      const int first = col % 32;
      for (int e = 0; e < 8; ++e) {
        const uint32_t c = (b[2 + (first + e) % 16] >> (first + e >= 16 ? 4 : 0)) & 15u;
        word |= (c ^ 8u) << (4 * nibble_of(e));
      }
      scale = static_cast<uint16_t>(b[0] | b[1] << 8);
    } else {
      const int g0 = col / a.w.group * a.w.group;
      const size_t base = static_cast<size_t>(row) * a.row_stride;
      float most = 0.f, mag = 0.f;
      bool bad = false;
      for (int c = g0; c < g0 + a.w.group; ++c) {
        const float v = ql::load_elem(a.dense, base + static_cast<size_t>(c) * a.col_stride, a.dtype);
        bad |= !isfinite(v);
        if (fabsf(v) > mag) {
          mag = fabsf(v);
          most = v;
        }
      }
      const __half hs = __float2half_rn(most / -8.0f);
      const float d = __half2float(hs);
      bad |= !isfinite(d);
      if (!bad && d != 0.f) {
        for (int e = 0; e < 8; ++e) {
          const float v =
              ql::load_elem(a.dense, base + static_cast<size_t>(col + e) * a.col_stride, a.dtype);
          const float q = fminf(fmaxf(rintf(v / d), -8.f), 7.f);
          word |= (static_cast<uint32_t>(static_cast<int>(q)) & 15u) << (4 * nibble_of(e));
        }
      }
      scale = bad ? 0x7fff : d == 0.f ? 0 : __half_as_ushort(hs);
    }
  }
  a.w.codes[id] = word;
  // one lane of the quad writes, where the group (or its padding) starts
  if ((lane & 3) == 0 && col % a.w.group == 0)
    reinterpret_cast<uint16_t*>(
        a.w.scales)[scale_at(a.w.group, a.w.chunks, tile, chunk, lane >> 2, i >> 1, i & 1)] = scale;
}

// The device order back to codes and scales (one thread per word).
__global__ void __launch_bounds__(256) q4_unpack_kernel(Q4View w, uint8_t* codes, uint16_t* scales) {
  const size_t id = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  const size_t per_tile = static_cast<size_t>(w.chunks) * 128;
  if (id >= per_tile * w.tiles) return;
  const size_t tile = id / per_tile;
  const int rest = static_cast<int>(id % per_tile);
  const int chunk = rest >> 7, lane = rest >> 2 & 31, i = rest & 3;
  int row, col;
  word_place(tile, chunk, lane, i, row, col);
  if (row >= w.n || col >= w.k) return;
  const uint32_t word = w.codes[id] ^ 0x88888888u;
  if (codes) {
    uint8_t* p = codes + (static_cast<size_t>(row) * w.k + col) / 2;
    for (int b = 0; b < 4; ++b)
      p[b] = static_cast<uint8_t>((word >> (4 * nibble_of(2 * b)) & 15u) |
                                  (word >> (4 * nibble_of(2 * b + 1)) & 15u) << 4);
  }
  if (scales && col % w.group == 0)
    scales[static_cast<size_t>(row) * (w.k / w.group) + col / w.group] =
        reinterpret_cast<const uint16_t*>(
            w.scales)[scale_at(w.group, w.chunks, tile, chunk, lane >> 2, i >> 1, i & 1)];
}

// An empty launch behind every write of a weight.  A product reads weights ahead of its
// griddepcontrol.wait, so that a write must have ended, its bytes visible, before the
// launch in front of the product begins.  This one, an ordinary launch, begins then; and
// whatever else stands between the write and a product (an event on another stream, a
// captured graph's edge, another kernel) waits for it in the same way.
__global__ void q4_written_kernel() {}

int close_write(ql_q4* w) {
  q4_written_kernel<<<1, 1, 0, w->ctx->stream>>>();
  QLN_CUDA(cudaGetLastError(), "launch behind the 4-bit layout");
  return QL_OK;
}

template <int FROM>
int launch_pack(ql_q4* w, PackArgs a) {
  a.w = view_of(w);
  const size_t blocks = (q4_words(w) + 255) / 256;
  q4_pack_kernel<FROM><<<static_cast<unsigned>(blocks), 256, 0, w->ctx->stream>>>(a);
  QLN_CUDA(cudaGetLastError(), "launch the 4-bit layout");
  return close_write(w);
}

// Device copies of host buffers for the length of one call.
struct Staged {
  ql_ctx* c;
  void* p[2] = {nullptr, nullptr};
  explicit Staged(ql_ctx* ctx) : c(ctx) {}
  ~Staged() {
    if (p[0] || p[1]) cudaStreamSynchronize(c->stream);
    for (void* q : p)
      if (q) cudaFree(q);
  }
  int copy(int slot, const void* host, size_t bytes) {
    QLN_CUDA(cudaMalloc(&p[slot], std::max<size_t>(bytes, 16)), "allocate a staging buffer");
    if (host)
      QLN_CUDA(cudaMemcpyAsync(p[slot], host, bytes, cudaMemcpyHostToDevice, c->stream),
               "copy to the device");
    return QL_OK;
  }
};

int check_mem(int mem) {
  if (mem != QL_MEM_DEVICE && mem != QL_MEM_HOST)
    return ql_fail(QL_ERR_INVALID, "unknown memory kind %d", mem);
  return QL_OK;
}

// ----------------------------------------------------------------- products --

struct LinearArgs {
  Q4View w;
  const void* x;
  const __half* x_scale;
  void* y;
  int64_t x_stride, y_stride;
  int rows, in_dtype, out_dtype;
};

// ---- the tensor-core product ----
// Formula: y[r][n] = sum over blocks of 32 columns of scale * (sum of (code - 8) x).
// The weights' bytes (0.52-0.56 of them per weight) are the cost of a few rows, so
// each goes from HBM to the lane that multiplies it once, through a ring in shared
// memory that every warp keeps for itself (cp.async, kD sets deep; a __syncwarp is
// the only barrier of the loop).  More than 32 rows (8 of f32) are passes, each with all
// of the weights.  Codes turn into f16 / bf16 exactly (a nibble in the
// mantissa of 1024 or 1/4, less an offset), or into int8 (a two's-complement nibble in
// the high half of a byte: 16 times its value).  The weights are the A operand (16
// rows of W), x the B operand (8 columns), so one row of x costs as much as eight.
// Blocks of 32 are summed on the tensor cores in f32 (int32 for Q8_0: exact), scaled
// in f32 and added to f32 sums.  f32 rows: three bf16 parts of 8 significand bits
// carry a value's 24 exactly (down to 2^-110, where the last part meets bf16's smallest
// step, 2^-133); the parts are three columns of B, whose sums are added at the end.
// One CTA an SM, each with an equal share of W's row tiles (with CTAs of a few tiles,
// several an SM, the last of them worked alone).  The columns are cut into 8 ranges, one for each warp of
// a team; WR teams take every WR-th tile.  The loads of the next tiles are under way
// while the ranges are joined, in order.  Every order of additions is the same for
// all variants and row counts, so a row's bits depend only on it and W.
constexpr int kRanges = 8;

// D = A B + C of one m16n8k16 (FIRST: D = A B).  Not volatile: the compiler
// interleaves the independent products of a chunk, which hides their latency.
template <bool BF, bool FIRST>
__device__ __forceinline__ void mma_f(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1) {
  const float c0 = FIRST ? 0.f : d[0], c1 = FIRST ? 0.f : d[1], c2 = FIRST ? 0.f : d[2],
              c3 = FIRST ? 0.f : d[3];
  if constexpr (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2),
          "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2),
          "f"(c3));
}

// D = A B + c of one m16n8k32 with the same addend everywhere.
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint4& a, uint32_t b0, uint32_t b1,
                                       int c) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%10,%10,%10,%10};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "r"(c));
}

// Asynchronous copies of this lane's bytes into shared memory; the first `bytes`
// of them are read, the rest are zeros.
__device__ __forceinline__ void cp16_stream(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(bytes)
               : "memory");
}
template <int N>
__device__ __forceinline__ void cp_cached(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void lds(uint32_t (&v)[N], uint32_t a) {
  static_assert(N == 1 || N == 2 || N == 4, "one access");
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(a));
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(a));
}
// Two f32 operations in one instruction, each rounded as by itself.
__device__ __forceinline__ uint64_t bits2(float2 v) {
  return static_cast<uint64_t>(__float_as_uint(v.y)) << 32 | __float_as_uint(v.x);
}
__device__ __forceinline__ float2 pair2(uint64_t v) {
  return make_float2(__uint_as_float(static_cast<uint32_t>(v)),
                     __uint_as_float(static_cast<uint32_t>(v >> 32)));
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return pair2(d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return pair2(d);
}

// (a & b) ^ c
__device__ __forceinline__ uint32_t and_xor(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// A word's eight values as four pairs in x's order, exactly; in bf16 2^-9 of them (an
// exponent is free to choose), so that a sum of 64 columns is no larger than the largest
// |x|: f32 and bf16 rows reach f32's largest numbers.
constexpr float kBfCodes = 512.f;
template <bool BF>
__device__ __forceinline__ void unpack_word(uint32_t w, uint32_t (&p)[4]) {
  if constexpr (BF) {
    const uint32_t in[4] = {w, w >> 8, w >> 4, w >> 12};
    const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x3e88),
                                                  __ushort_as_bfloat16(0x3e88));  // 136 / 512
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t h = and_xor(in[i], 0x000f000fu, 0x3e883e88u);  // (128 + (value + 8)) / 512
      const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&h), off);
      p[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  } else {
    const __half2 off = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));  // 1032
    const __half2 s16 = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00));  // 1/16
    const __half2 m72 = __halves2half2(__ushort_as_half(0xd480), __ushort_as_half(0xd480));  // -72
    const uint32_t in[2] = {w, w >> 8};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t lo = and_xor(in[i], 0x000f000fu, 0x64086408u);  // 1024 + (value + 8)
      const uint32_t hi = and_xor(in[i], 0x00f000f0u, 0x64806480u);  // 1024 + 16 (value + 8)
      const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), off);
      const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&hi), s16, m72);
      p[i] = *reinterpret_cast<const uint32_t*>(&a);
      p[i + 2] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
}

template <int IN, int NT, int MT, int WR, int G>
struct LinCfg {
  static constexpr bool kQ8 = IN == ql::kQ8_0;
  static constexpr bool kBF = IN == ql::kBF16 || IN == ql::kF32;
  static constexpr int kParts = IN == ql::kF32 ? 3 : 1;
  static constexpr int kTileRows = IN == ql::kF32 ? 2 : 8;  // rows of x in 8 columns of B
  static constexpr int kRows = NT * kTileRows;              // and in one pass
  static constexpr int kWarps = kRanges * WR, kThreads = 32 * kWarps;
  static constexpr int kGroup = MT * WR;  // tiles that the CTA works on at a time
  // one set of a warp: MT tiles of codes, their scales, 64 columns of x's rows
  static constexpr int kScaleTile = G == 32 ? 64 : 32;
  static constexpr int kXRow = kQ8 ? 64 : IN == ql::kF32 ? 256 : 128;
  static constexpr int kScales = MT * 512;
  static constexpr int kX = kScales + MT * kScaleTile;
  static constexpr int kXScales = kX + kRows * kXRow;  // Q8_0: two f16 a row
  static constexpr int kSet = kXScales + (kQ8 ? kRows * 4 : 0);
  static constexpr int kPitch = 16 * kGroup + 4;  // of a column in the join
  static constexpr int kJoin = 8 * kPitch * 4;    // a range's 8 columns
  static constexpr int kRoom = 227 * 1024 - kRanges * kJoin;
  static constexpr int kD = 4 * kWarps * kSet <= kRoom ? 4 : 3 * kWarps * kSet <= kRoom ? 3 : 2;
  static constexpr int kRing = kWarps * kD * kSet;
  static constexpr int kSmem = kRing + kRanges * kJoin;
};

template <int IN, int NT, int MT, int WR, int G>
__global__ void __launch_bounds__(kRanges* WR * 32, 1) linear_q4_kernel(const LinearArgs a) {
  using C = LinCfg<IN, NT, MT, WR, G>;
  extern __shared__ __align__(16) char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int range = warp % kRanges, team = warp / kRanges;
  const int r0 = blockIdx.y * C::kRows;
  const int rows = min(a.rows - r0, C::kRows);
  const int chunks = a.w.chunks, K = a.w.k;
  // this CTA's tiles [t0, t1) and this warp's chunks [c0, c0 + nc)
  const int t0 = static_cast<int>(static_cast<long long>(a.w.tiles) * blockIdx.x / gridDim.x);
  const int t1 = static_cast<int>(static_cast<long long>(a.w.tiles) * (blockIdx.x + 1) / gridDim.x);
  const int groups = (t1 - t0 + C::kGroup - 1) / C::kGroup;
  const int c0 = static_cast<int>(static_cast<long long>(chunks) * range / kRanges);
  const int nc = static_cast<int>(static_cast<long long>(chunks) * (range + 1) / kRanges) - c0;

  const uint32_t ring = ql::smem_u32(smem) + warp * C::kD * C::kSet;
  const uint32_t join = ql::smem_u32(smem) + C::kRing;
  // tiles of this team in a group: first, first + WR, ... below t1
  auto live_tiles = [&](int group) {
    const int left = t1 - (t0 + group * C::kGroup + team);
    return left <= 0 ? 0 : min(MT, (left + WR - 1) / WR);
  };
  // ---- loads: where the next set's weights lie (advanced chunk by chunk)
  const uint32_t wstep = static_cast<uint32_t>(WR) * chunks * 512u;  // tile to tile of the team
  constexpr int kLanes = C::kScaleTile / 16;  // lanes that copy a tile's scales, 16 bytes each
  const char* wp;
  const char* sp;
  int lg = 0, lc = c0, llive = 0;  // group and chunk of the next set
  auto start_group = [&](int group) {
    const size_t tile = t0 + group * C::kGroup + team;
    wp = reinterpret_cast<const char*>(a.w.codes) + (tile * chunks + c0) * 512 + lane * 16;
    sp = reinterpret_cast<const char*>(a.w.scales) +
         scale_at(G, chunks, tile + lane / kLanes * WR, 0, 0, 0, 0) * 2 + lane % kLanes * 16;
    llive = live_tiles(group);
  };
  start_group(0);
  auto copy_w = [&](uint32_t set) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
      if (m < llive) cp16_stream(set + m * 512 + lane * 16, wp + m * wstep, 16);
    if (lane < llive * kLanes)
      cp_cached<16>(set + C::kScales + lane * 16,
                    sp + (G == 32 ? lc * 64 : G == 64 ? lc * 32 : (lc >> 1) * 32), 16);
  };
  auto next = [&]() {
    wp += 512;
    if (++lc == c0 + nc) {
      lc = c0;
      start_group(++lg);
    }
  };
  // x: 16-byte units of a row's 64 columns, spread so that the lanes of a fragment
  // read from different banks.  Rows past the call's are left as they are: their
  // columns of the product are not stored.
  constexpr int kBytes = IN == ql::kF32 ? 4 : C::kQ8 ? 1 : 2;
  constexpr int kUnits = C::kXRow / 16;  // of a row: 4, 8 or 16
  constexpr int kXU = (C::kRows * kUnits + 31) / 32;
  const bool vec =
      (reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.x_stride * kBytes)) % 16 == 0;
  auto unit_at = [](int r, int u) {
    if constexpr (C::kQ8) return r * C::kXRow + (u ^ (r & 2)) * 16;
    else if constexpr (IN == ql::kF32) return r * C::kXRow + (u ^ (r & 1)) * 16;
    else return r * C::kXRow + (u ^ (r & 1) * 4) * 16;
  };
  // this lane's units: column xcol of rows xr, xr + 32 / kUnits, ...
  const int xr = lane / kUnits, xcol = lane % kUnits * (16 / kBytes);
  const char* const xp = static_cast<const char*>(a.x) +
                         (static_cast<size_t>(r0 + xr) * a.x_stride + xcol) * kBytes;
  const size_t xstep = static_cast<size_t>(32 / kUnits) * a.x_stride * kBytes;
  // (rows 32 / kUnits apart are spread alike: their places are 512 bytes apart)
  const uint32_t xdst = C::kX + unit_at(xr, lane % kUnits);
  // Q8_0: the scales of x's row `lane`, two of a chunk at a time
  const uint16_t* const xsp =
      reinterpret_cast<const uint16_t*>(a.x_scale) + static_cast<size_t>(r0 + lane) * (K / 32);
  const bool xs_vec = C::kQ8 && (reinterpret_cast<uintptr_t>(a.x_scale) | (K / 32 * 2)) % 4 == 0;
  auto copy_x = [&](uint32_t set, int c) {
    const char* const p = xp + c * (64 * kBytes);
    if (vec && 64 * c + 64 <= K) {
#pragma unroll
      for (int i = 0; i < kXU; ++i)
        if (xr + i * (32 / kUnits) < rows) cp_cached<16>(set + xdst + 512 * i, p + i * xstep, 16);
    } else {  // the last half chunk, or rows that do not start on 16 bytes
      const bool in = 64 * c + xcol < K;
#pragma unroll 1
      for (int i = 0; i < kXU; ++i) {
        if (xr + i * (32 / kUnits) >= rows) break;
        const char* const q = p + i * xstep;
        uint32_t v[4] = {0, 0, 0, 0};
        if (in) {
#pragma unroll
          for (int e = 0; e < 16 / kBytes; ++e) {
            if constexpr (IN == ql::kF32) v[e] = reinterpret_cast<const uint32_t*>(q)[e];
            else if constexpr (C::kQ8)
              v[e / 4] |= static_cast<uint32_t>(reinterpret_cast<const uint8_t*>(q)[e])
                          << (8 * (e % 4));
            else
              v[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(q)[e])
                          << (16 * (e % 2));
          }
        }
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(set + xdst + 512 * i), "r"(v[0]),
                     "r"(v[1]), "r"(v[2]), "r"(v[3])
                     : "memory");
      }
    }
    if constexpr (C::kQ8) {
      if (lane < rows) {
        if (xs_vec) {
          cp_cached<4>(set + C::kXScales + lane * 4, xsp + 2 * c, 4);
        } else {
          const uint32_t v =
              xsp[2 * c] | (64 * c + 32 < K ? static_cast<uint32_t>(xsp[2 * c + 1]) << 16 : 0u);
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(set + C::kXScales + lane * 4), "r"(v)
                       : "memory");
        }
      }
    }
  };
  // ---- products
  // f32: this lane's column is part g % 3 of row g / 3; the bits that parts 1 and 2
  // take off first
  const int part = g % 3;
  const uint32_t m1 = part >= 1 ? 0xffff0000u : 0u, m2 = part == 2 ? 0xffff0000u : 0u;
  // The fragment of block j in B tile q: eight values of this lane's column.
  auto fragment = [&](uint32_t set, int q, int j, uint32_t (&o)[C::kQ8 ? 2 : 4]) {
    if constexpr (IN == ql::kF32) {
      const int r = 2 * q + min(g / 3, 1);
      uint32_t f[2][4];
      lds(f[0], set + C::kX + unit_at(r, 8 * j + 2 * t));
      lds(f[1], set + C::kX + unit_at(r, 8 * j + 2 * t + 1));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = __uint_as_float(f[h][e]);
          v -= __uint_as_float(__float_as_uint(v) & m1);
          v -= __uint_as_float(__float_as_uint(v) & m2);
          f[h][e] = __float_as_uint(v);
        }
        o[2 * h] = __byte_perm(f[h][0], f[h][1], 0x7632);
        o[2 * h + 1] = __byte_perm(f[h][2], f[h][3], 0x7632);
      }
    } else if constexpr (C::kQ8) {
      lds(o, set + C::kX + unit_at(8 * q + g, 2 * j + t / 2) + t % 2 * 8);
      o[0] = __byte_perm(o[0], 0, 0x3120);  // the order of the codes' bytes
      o[1] = __byte_perm(o[1], 0, 0x3120);
    } else {
      lds(o, set + C::kX + unit_at(8 * q + g, 4 * j + t));
    }
  };
  float2 acc[MT][NT][2];  // [rows g, g + 8]: columns 2t, 2t + 1
  uint32_t x[NT][2][C::kQ8 ? 2 : 4];
  float2 xs[C::kQ8 ? NT : 1][2];  // Q8_0: [block], of columns 2t, 2t + 1
  auto product = [&](uint32_t set, int m) {
    uint32_t w[4], sr[G == 32 ? 2 : 1];
    lds(w, set + m * 512 + lane * 16);
    lds(sr, set + C::kScales + m * C::kScaleTile + g * (C::kScaleTile / 8));
    float2 s[2];  // rows g, g + 8
    s[0] = __half22float2(*reinterpret_cast<const __half2*>(&sr[0]));
    s[1] = __half22float2(*reinterpret_cast<const __half2*>(&sr[G == 32 ? 1 : 0]));
    if constexpr (C::kQ8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint4 A = make_uint4((w[2 * j] << 4) & 0xf0f0f0f0u, (w[2 * j + 1] << 4) & 0xf0f0f0f0u,
                                   w[2 * j] & 0xf0f0f0f0u, w[2 * j + 1] & 0xf0f0f0f0u);
#pragma unroll
        for (int q = 0; q < NT; ++q) {
          // sums start at the bits of 1.5 * 2^23: below 2^22 they are the
          // mantissa of a float, and a subtraction converts them
          int d[4];
          mma_s8(d, A, x[q][j][0], x[q][j][1], 0x4b400000);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float sh = h ? s[j].y : s[j].x;
            const float2 f = add2(make_float2(__int_as_float(d[2 * h]), __int_as_float(d[2 * h + 1])),
                                  make_float2(-12582912.0f, -12582912.0f));
            acc[m][q][h] = fma2(f, mul2(make_float2(sh, sh), xs[q][j]), acc[m][q][h]);
          }
        }
      }
    } else {
      float d[NT][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t lo[4], hi[4];  // rows g and g + 8
        unpack_word<C::kBF>(w[2 * j], lo);
        unpack_word<C::kBF>(w[2 * j + 1], hi);
        const uint32_t A0[4] = {lo[0], hi[0], lo[1], hi[1]};
        const uint32_t A1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
        for (int q = 0; q < NT; ++q) {
          if (G == 32 || j == 0) mma_f<C::kBF, true>(d[q], A0, x[q][j][0], x[q][j][1]);
          else mma_f<C::kBF, false>(d[q], A0, x[q][j][0], x[q][j][1]);
        }
#pragma unroll
        for (int q = 0; q < NT; ++q) mma_f<C::kBF, false>(d[q], A1, x[q][j][2], x[q][j][3]);
        if (G == 32 || j == 1) {
#pragma unroll
          for (int q = 0; q < NT; ++q) {
            acc[m][q][0] =
                fma2(make_float2(d[q][0], d[q][1]), make_float2(s[j].x, s[j].x), acc[m][q][0]);
            acc[m][q][1] =
                fma2(make_float2(d[q][2], d[q][3]), make_float2(s[j].y, s[j].y), acc[m][q][1]);
          }
        }
      }
    }
  };

  // The first weights do not depend on the kernel before this one (an empty launch
  // stands between a write of them and any product).
  const int total = groups * nc;
#pragma unroll
  for (int i = 0; i < C::kD - 1; ++i)
    if (i < total) {
      copy_w(ring + i * C::kSet);
      next();
    }
  ql::griddep_wait();
  ql::griddep_launch_dependents();
#pragma unroll
  for (int i = 0; i < C::kD - 1; ++i) {
    if (i < total) copy_x(ring + i * C::kSet, c0 + i % nc);
    cp_commit();
  }
  uint32_t set = ring, load_set = ring + (C::kD - 1) * C::kSet;
  const uint32_t ring_end = ring + C::kD * C::kSet;
  int to_load = total - (C::kD - 1);
  for (int group = 0; group < groups; ++group) {
    const int live = live_tiles(group);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int q = 0; q < NT; ++q) acc[m][q][0] = acc[m][q][1] = make_float2(0.f, 0.f);
    for (int i = 0; i < nc; ++i) {
      cp_wait<C::kD - 2>();
      __syncwarp();  // the set has arrived for every lane, and the one before is read
      if (to_load > 0) {
        copy_w(load_set);
        copy_x(load_set, lc);
        next();
      }
      --to_load;
      cp_commit();
      load_set = load_set + C::kSet == ring_end ? ring : load_set + C::kSet;
#pragma unroll
      for (int q = 0; q < NT; ++q)
#pragma unroll
        for (int j = 0; j < 2; ++j) fragment(set, q, j, x[q][j]);
      if constexpr (C::kQ8) {
#pragma unroll
        for (int q = 0; q < NT; ++q) {
          uint32_t v[2];  // rows 8q + 2t and the next
          lds(v, set + C::kXScales + (8 * q + 2 * t) * 4);
          const float2 even = __half22float2(*reinterpret_cast<const __half2*>(&v[0]));
          const float2 odd = __half22float2(*reinterpret_cast<const __half2*>(&v[1]));
          xs[q][0] = make_float2(even.x, odd.x);
          xs[q][1] = make_float2(even.y, odd.y);
        }
      }
      if (live == MT) {
#pragma unroll
        for (int m = 0; m < MT; ++m) product(set, m);
      } else {
#pragma unroll
        for (int m = 0; m < MT - 1; ++m)
          if (m < live) product(set, m);
      }
      set = set + C::kSet == ring_end ? ring : set + C::kSet;
    }
    // Join the ranges, eight columns of B at a time: [range][column][row].
    const int n0 = (t0 + group * C::kGroup) * 16;
    const int n1 = min(min(C::kGroup * 16, t1 * 16 - n0), a.w.n - n0);
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      if (q * C::kTileRows >= rows) break;
      if (group > 0 || q > 0) __syncthreads();  // the sums before have been read
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m >= live) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(
                           join + range * C::kJoin +
                           ((2 * t + (i & 1)) * C::kPitch + 16 * (m * WR + team) + g +
                            8 * (i >> 1)) * 4),
                       "f"(i & 1 ? acc[m][q][i >> 1].y : acc[m][q][i >> 1].x)
                       : "memory");
      }
      __syncthreads();
      const int left = min(C::kTileRows, rows - q * C::kTileRows);
      for (int i = threadIdx.x; i < 16 * C::kGroup * left; i += C::kThreads) {
        const int row = i % (16 * C::kGroup), r = i / (16 * C::kGroup);
        if (row >= n1) continue;
        float y = 0.f;
#pragma unroll
        for (int p = C::kParts - 1; p >= 0; --p) {  // the small parts first
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < kRanges; ++w) {
            float z;
            asm volatile("ld.shared.f32 %0, [%1];"
                         : "=f"(z)
                         : "r"(join + w * C::kJoin + ((r * C::kParts + p) * C::kPitch + row) * 4)
                         : "memory");
            v += z;
          }
          y += v;
        }
        if (C::kQ8) y *= 0.0625f;  // the codes were 16 times their values
        if (C::kBF) y *= kBfCodes;
        ql::store_elem(a.y, static_cast<size_t>(r0 + q * C::kTileRows + r) * a.y_stride + n0 + row,
                       a.out_dtype, y);
      }
    }
  }
}

template <int IN, int NT, int MT, int WR, int G>
cudaError_t launch_linear_as(const LinearArgs& a, int num_sms, cudaStream_t s) {
  using C = LinCfg<IN, NT, MT, WR, G>;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  auto* const kernel = linear_q4_kernel<IN, NT, MT, WR, G>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = ql_once_per_device(done, [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  for (int64_t r = 0; e == cudaSuccess && r < a.rows; r += 65535 * C::kRows) {  // grid.y's limit
    LinearArgs b = a;
    b.rows = static_cast<int>(std::min<int64_t>(a.rows - r, 65535 * C::kRows));
    const size_t xb = type_bytes(a.in_dtype), yb = type_bytes(a.out_dtype);
    b.x = static_cast<const char*>(a.x) + static_cast<size_t>(r) * a.x_stride * xb;
    b.x_scale = a.x_scale ? a.x_scale + static_cast<size_t>(r) * (a.w.k / 32) : nullptr;
    b.y = static_cast<char*>(a.y) + static_cast<size_t>(r) * a.y_stride * yb;
    const dim3 grid(std::min(num_sms, a.w.tiles), (b.rows + C::kRows - 1) / C::kRows);
    e = launch_pdl(kernel, grid, dim3(C::kThreads), C::kSmem, s, b);
  }
  return e;
}

// B tiles by the rows of x.  Two teams of warps (16 warps hide more latency: 1 x 8192 ->
// 57344 f16 55 us, 59 us with one, both before later steps brought it to 52) unless the SMs have no second tile for the second
// team (1 x 2048 -> 2048 Q8_0 2.8 us with one team, 3.2 us with two).  With four B
// tiles the sums fill the registers of one team (32 x 8192 -> 28672 f16 64 us, 116 us
// with two teams of half the tiles), eight tiles at a time where a CTA has more than
// four (86 us with four at a time).
template <int IN, int G>
cudaError_t launch_linear_in(const LinearArgs& a, int num_sms, cudaStream_t s) {
  const int b = (a.rows - 1) / LinCfg<IN, 1, 1, 1, G>::kTileRows + 1;
  if (b > 2)
    return a.w.tiles <= 4 * num_sms ? launch_linear_as<IN, 4, 4, 1, G>(a, num_sms, s)
                                    : launch_linear_as<IN, 4, 8, 1, G>(a, num_sms, s);
  const bool one = a.w.tiles <= num_sms;
  if (b == 1)
    return one ? launch_linear_as<IN, 1, 1, 1, G>(a, num_sms, s)
               : launch_linear_as<IN, 1, 4, 2, G>(a, num_sms, s);
  return one ? launch_linear_as<IN, 2, 1, 1, G>(a, num_sms, s)
             : launch_linear_as<IN, 2, 4, 2, G>(a, num_sms, s);
}

cudaError_t launch_linear(const LinearArgs& a, int num_sms, cudaStream_t s) {
  auto by_group = [&](auto in) {
    constexpr int IN = decltype(in)::value;
    if (a.w.group == 32) return launch_linear_in<IN, 32>(a, num_sms, s);
    if (a.w.group == 64) return launch_linear_in<IN, 64>(a, num_sms, s);
    return launch_linear_in<IN, 128>(a, num_sms, s);
  };
  switch (a.in_dtype) {
    case QL_F32: return by_group(std::integral_constant<int, ql::kF32>());
    case QL_F16: return by_group(std::integral_constant<int, ql::kF16>());
    case QL_BF16: return by_group(std::integral_constant<int, ql::kBF16>());
    default: return by_group(std::integral_constant<int, ql::kQ8_0>());
  }
}

}  // namespace

// Quantises element (row, col) = dense[row * row_stride + col * col_stride] on
// the context's stream (ql_llama_quantize reads its transposed weights this way).
int ql_q4_quantize_strided(ql_q4* w, const void* dense, int dtype, int64_t row_stride,
                           int64_t col_stride) {
  PackArgs a{};
  a.dense = dense;
  a.dtype = dtype;
  a.row_stride = row_stride;
  a.col_stride = col_stride;
  return launch_pack<kPackDense>(w, a);
}

extern "C" {

int ql_rms_norm(ql_ctx* c, const ql_norm_args* args) {
  if (!c || !args) return ql_fail(QL_ERR_INVALID, "ql_rms_norm: NULL argument");
  const ql_norm_args& f = *args;
  if (f.rows < 0) return ql_fail(QL_ERR_INVALID, "row count %d is negative", f.rows);
  if (f.hidden <= 0) return ql_fail(QL_ERR_INVALID, "hidden must be positive, got %d", f.hidden);
  if (f.hidden > (1 << 30)) return ql_fail(QL_ERR_UNSUPPORTED, "hidden %d is too large", f.hidden);
  if (!float_type(f.in_dtype) || !float_type(f.weight_dtype) ||
      !(float_type(f.out_dtype) || f.out_dtype == QL_Q8_0))
    return ql_fail(QL_ERR_INVALID, "unsupported element types %d, %d -> %d", f.in_dtype,
                   f.weight_dtype, f.out_dtype);
  if (!std::isfinite(f.eps) || f.eps < 0.f)
    return ql_fail(QL_ERR_INVALID, "RMSNorm eps must be finite and nonnegative");
  if (f.out_dtype == QL_Q8_0 && f.hidden % 32 != 0)
    return ql_fail(QL_ERR_INVALID, "a Q8_0 output needs hidden divisible by 32, got %d", f.hidden);
  if (f.sum_out && !f.residual)
    return ql_fail(QL_ERR_INVALID, "ql_rms_norm: sum_out needs a residual");
  const int64_t xs = f.x_stride ? f.x_stride : f.hidden;
  const int64_t rs = f.residual_stride ? f.residual_stride : f.hidden;
  if (xs < f.hidden || (f.residual && rs < f.hidden))
    return ql_fail(QL_ERR_INVALID, "a row stride is smaller than hidden %d", f.hidden);
  if (f.rows == 0) return QL_OK;
  if (!f.x || !f.weight || !f.out || (f.out_dtype == QL_Q8_0 && !f.out_scale))
    return ql_fail(QL_ERR_INVALID, "ql_rms_norm: NULL buffer");
  const size_t ib = type_bytes(f.in_dtype);
  if (!aligned(f.x, ib) || !aligned(f.residual, ib) || !aligned(f.sum_out, ib) ||
      !aligned(f.weight, type_bytes(f.weight_dtype)) || !aligned(f.out, type_bytes(f.out_dtype)) ||
      !aligned(f.out_scale, 2))
    return ql_fail(QL_ERR_INVALID, "ql_rms_norm: a buffer is not aligned to its element size");
  // Outputs may be inputs, element on element, and nothing else may overlap.
  struct Span {
    const char* p;
    size_t bytes;
    int64_t stride;
    int dtype;
  };
  auto span = [&](const void* p, int64_t stride, int dt) {
    const size_t n = static_cast<size_t>(stride) * (f.rows - 1) + f.hidden;
    return Span{static_cast<const char*>(p), p ? n * type_bytes(dt) : 0, f.rows > 1 ? stride : 0, dt};
  };
  auto clash = [](const Span& a, const Span& b, bool same) {
    if (!a.bytes || !b.bytes || a.p >= b.p + b.bytes || b.p >= a.p + a.bytes) return false;
    return !(same && a.p == b.p && a.stride == b.stride && a.dtype == b.dtype);
  };
  const Span in[] = {span(f.x, xs, f.in_dtype), span(f.residual, rs, f.in_dtype)};
  const Span w{static_cast<const char*>(f.weight), f.hidden * type_bytes(f.weight_dtype), 0, -1};
  const Span outs[] = {span(f.sum_out, f.hidden, f.in_dtype), span(f.out, f.hidden, f.out_dtype),
                       Span{static_cast<const char*>(f.out_scale),
                            f.out_dtype == QL_Q8_0 ? static_cast<size_t>(f.rows) * (f.hidden / 32) * 2 : 0,
                            0, -1}};
  bool bad = clash(outs[0], outs[1], false) || clash(outs[0], outs[2], false) ||
             clash(outs[1], outs[2], false);
  for (const Span& o : outs) bad |= clash(o, w, false) || clash(o, in[0], true) || clash(o, in[1], true);
  if (bad) return ql_fail(QL_ERR_INVALID, "ql_rms_norm: an output overlaps another buffer");
  ql_device_guard dev(c->device);
  QLN_CUDA(dev.error(), "set device");
  NormArgs a{};
  a.x = f.x;
  a.residual = f.residual;
  a.weight = f.weight;
  a.sum_out = f.sum_out;
  a.out = f.out;
  a.out_scale = static_cast<__half*>(f.out_scale);
  a.x_stride = xs;
  a.residual_stride = rs;
  a.rows = f.rows;
  a.hidden = f.hidden;
  a.inv_hidden = 1.0f / static_cast<float>(f.hidden);
  a.in_dtype = f.in_dtype;
  a.weight_dtype = f.weight_dtype;
  a.out_dtype = f.out_dtype;
  a.eps = f.eps;
  QLN_CUDA(launch_norm(a, c->num_sms, c->stream), "launch rms_norm");
  return QL_OK;
}

int ql_q4_create(ql_ctx* c, int32_t out_features, int32_t in_features, int32_t group,
                 ql_q4** out) {
  if (!c || !out) return ql_fail(QL_ERR_INVALID, "ql_q4_create: NULL argument");
  *out = nullptr;
  if (out_features <= 0 || in_features <= 0)
    return ql_fail(QL_ERR_INVALID, "weight dimensions must be positive, got [%d, %d]",
                   out_features, in_features);
  if (group != 32 && group != 64 && group != 128)
    return ql_fail(QL_ERR_INVALID, "group %d must be 32, 64 or 128", group);
  if (in_features % group != 0)
    return ql_fail(QL_ERR_INVALID, "in_features %d must be divisible by the group %d", in_features,
                   group);
  if (out_features > (1 << 30) || in_features > (1 << 24))
    return ql_fail(QL_ERR_UNSUPPORTED, "weight dimensions [%d, %d] are too large", out_features,
                   in_features);
  ql_device_guard dev(c->device);
  QLN_CUDA(dev.error(), "set device");
  ql_q4* w = new (std::nothrow) ql_q4;
  if (!w) return ql_fail(QL_ERR_OOM, "ql_q4_create: out of host memory");
  w->ctx = c;
  w->n = out_features;
  w->k = in_features;
  w->group = group;
  w->tiles = (out_features + 15) / 16;
  w->chunks = (in_features + 63) / 64;
  cudaError_t e = cudaMalloc(&w->codes, q4_words(w) * 4);
  if (e == cudaSuccess) e = cudaMalloc(&w->scales, q4_scales(w) * 2);
  // a handle without values yet multiplies by zero
  if (e == cudaSuccess) e = cudaMemsetAsync(w->codes, 0, q4_words(w) * 4, c->stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(w->scales, 0, q4_scales(w) * 2, c->stream);
  if (e != cudaSuccess) {
    ql_q4_destroy(w);
    cudaGetLastError();
    return ql_fail(e == cudaErrorMemoryAllocation ? QL_ERR_OOM : QL_ERR_CUDA,
                   "allocate a 4-bit weight: %s", cudaGetErrorString(e));
  }
  if (int r = close_write(w)) {
    ql_q4_destroy(w);
    return r;
  }
  *out = w;
  return QL_OK;
}

int ql_q4_destroy(ql_q4* w) {
  if (!w) return QL_OK;
  ql_device_guard dev(w->ctx->device);
  cudaStreamSynchronize(w->ctx->stream);
  if (w->codes) cudaFree(w->codes);
  if (w->scales) cudaFree(w->scales);
  delete w;
  return QL_OK;
}

int ql_q4_shape(const ql_q4* w, int32_t* out_features, int32_t* in_features, int32_t* group) {
  if (!w || !out_features || !in_features || !group)
    return ql_fail(QL_ERR_INVALID, "ql_q4_shape: NULL argument");
  *out_features = w->n;
  *in_features = w->k;
  *group = w->group;
  return QL_OK;
}

int ql_q4_set(ql_q4* w, const uint8_t* codes, const void* scales, int32_t mem) {
  if (!w || !codes || !scales) return ql_fail(QL_ERR_INVALID, "ql_q4_set: NULL argument");
  if (int r = check_mem(mem)) return r;
  if (!aligned(scales, 2)) return ql_fail(QL_ERR_INVALID, "ql_q4_set: scales are not aligned");
  ql_device_guard dev(w->ctx->device);
  QLN_CUDA(dev.error(), "set device");
  PackArgs a{};
  a.bytes = codes;
  a.scales = static_cast<const uint16_t*>(scales);
  if (mem == QL_MEM_DEVICE) return launch_pack<kPackCodes>(w, a);
  Staged s(w->ctx);
  const size_t nk = static_cast<size_t>(w->n) * w->k;
  if (int r = s.copy(0, codes, nk / 2)) return r;
  if (int r = s.copy(1, scales, nk / w->group * 2)) return r;
  a.bytes = static_cast<const uint8_t*>(s.p[0]);
  a.scales = static_cast<const uint16_t*>(s.p[1]);
  return launch_pack<kPackCodes>(w, a);
}

int ql_q4_set_blocks(ql_q4* w, const void* blocks, int64_t bytes, int32_t mem) {
  if (!w || !blocks) return ql_fail(QL_ERR_INVALID, "ql_q4_set_blocks: NULL argument");
  if (int r = check_mem(mem)) return r;
  if (w->group != 32)
    return ql_fail(QL_ERR_INVALID, "Q4_0 blocks need a group of 32, the weight has %d", w->group);
  const int64_t want = static_cast<int64_t>(w->n) * (w->k / 32) * 18;
  if (bytes != want)
    return ql_fail(QL_ERR_INVALID, "Q4_0 blocks of [%d, %d] take %lld bytes, got %lld", w->n, w->k,
                   (long long)want, (long long)bytes);
  ql_device_guard dev(w->ctx->device);
  QLN_CUDA(dev.error(), "set device");
  PackArgs a{};
  a.bytes = static_cast<const uint8_t*>(blocks);
  if (mem == QL_MEM_DEVICE) return launch_pack<kPackBlocks>(w, a);
  Staged s(w->ctx);
  if (int r = s.copy(0, blocks, static_cast<size_t>(bytes))) return r;
  a.bytes = static_cast<const uint8_t*>(s.p[0]);
  return launch_pack<kPackBlocks>(w, a);
}

int ql_q4_quantize(ql_q4* w, const void* dense, int32_t dtype, int64_t row_stride, int32_t mem) {
  if (!w || !dense) return ql_fail(QL_ERR_INVALID, "ql_q4_quantize: NULL argument");
  if (int r = check_mem(mem)) return r;
  if (!float_type(dtype)) return ql_fail(QL_ERR_INVALID, "unsupported element type %d", dtype);
  const int64_t rs = row_stride ? row_stride : w->k;
  if (rs < w->k)
    return ql_fail(QL_ERR_INVALID, "a row stride is smaller than in_features %d", w->k);
  if (!aligned(dense, type_bytes(dtype)))
    return ql_fail(QL_ERR_INVALID, "ql_q4_quantize: the matrix is not aligned to its element size");
  ql_device_guard dev(w->ctx->device);
  QLN_CUDA(dev.error(), "set device");
  if (mem == QL_MEM_DEVICE) return ql_q4_quantize_strided(w, dense, dtype, rs, 1);
  Staged s(w->ctx);
  const size_t elems = static_cast<size_t>(rs) * (w->n - 1) + w->k;
  if (int r = s.copy(0, dense, elems * type_bytes(dtype))) return r;
  return ql_q4_quantize_strided(w, s.p[0], dtype, rs, 1);
}

int ql_q4_get(const ql_q4* w, uint8_t* codes, void* scales, int32_t mem) {
  if (!w) return ql_fail(QL_ERR_INVALID, "ql_q4_get: NULL argument");
  if (int r = check_mem(mem)) return r;
  if (!aligned(scales, 2)) return ql_fail(QL_ERR_INVALID, "ql_q4_get: scales are not aligned");
  ql_device_guard dev(w->ctx->device);
  QLN_CUDA(dev.error(), "set device");
  cudaStream_t st = w->ctx->stream;
  const size_t cb = static_cast<size_t>(w->n) * w->k / 2;
  const size_t sb = static_cast<size_t>(w->n) * (w->k / w->group) * 2;
  Staged s(w->ctx);
  uint8_t* dc = codes;
  void* ds = scales;
  if (mem == QL_MEM_HOST) {
    if (codes) {
      if (int r = s.copy(0, nullptr, cb)) return r;
      dc = static_cast<uint8_t*>(s.p[0]);
    }
    if (scales) {
      if (int r = s.copy(1, nullptr, sb)) return r;
      ds = s.p[1];
    }
  }
  const size_t blocks = (q4_words(w) + 255) / 256;
  q4_unpack_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(view_of(w), dc,
                                                                  static_cast<uint16_t*>(ds));
  QLN_CUDA(cudaGetLastError(), "launch the 4-bit read-back");
  if (mem == QL_MEM_HOST) {
    if (codes) QLN_CUDA(cudaMemcpyAsync(codes, dc, cb, cudaMemcpyDeviceToHost, st), "copy codes");
    if (scales)
      QLN_CUDA(cudaMemcpyAsync(scales, ds, sb, cudaMemcpyDeviceToHost, st), "copy scales");
  }
  return QL_OK;
}

int ql_linear_q4(ql_ctx* c, const ql_q4* w, const ql_linear_args* args) {
  if (!c || !w || !args) return ql_fail(QL_ERR_INVALID, "ql_linear_q4: NULL argument");
  const ql_linear_args& f = *args;
  if (w->ctx->device != c->device)
    return ql_fail(QL_ERR_INVALID, "the weight lives on device %d, the context on device %d",
                   w->ctx->device, c->device);
  if (f.rows < 0) return ql_fail(QL_ERR_INVALID, "row count %d is negative", f.rows);
  if (!(float_type(f.in_dtype) || f.in_dtype == QL_Q8_0) || !float_type(f.out_dtype))
    return ql_fail(QL_ERR_INVALID, "unsupported element types %d -> %d", f.in_dtype, f.out_dtype);
  const int64_t xs = f.x_stride ? f.x_stride : w->k, ys = f.y_stride ? f.y_stride : w->n;
  if (xs < w->k || ys < w->n)
    return ql_fail(QL_ERR_INVALID, "a row stride is smaller than the row (%d in, %d out)", w->k,
                   w->n);
  if (f.rows == 0) return QL_OK;
  if (!f.x || !f.y || (f.in_dtype == QL_Q8_0 && !f.x_scale))
    return ql_fail(QL_ERR_INVALID, "ql_linear_q4: NULL buffer");
  if (!aligned(f.x, type_bytes(f.in_dtype)) || !aligned(f.y, type_bytes(f.out_dtype)) ||
      !aligned(f.x_scale, 2))
    return ql_fail(QL_ERR_INVALID, "ql_linear_q4: a buffer is not aligned to its element size");
  ql_device_guard dev(c->device);
  QLN_CUDA(dev.error(), "set device");
  LinearArgs a{};
  a.w = view_of(w);
  a.x = f.x;
  a.x_scale = static_cast<const __half*>(f.x_scale);
  a.y = f.y;
  a.x_stride = xs;
  a.y_stride = ys;
  a.rows = f.rows;
  a.in_dtype = f.in_dtype;
  a.out_dtype = f.out_dtype;
  QLN_CUDA(launch_linear(a, c->num_sms, c->stream), "launch the 4-bit product");
  return QL_OK;
}

}  // extern "C"
