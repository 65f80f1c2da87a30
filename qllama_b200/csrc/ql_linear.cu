// ql_linear.cu -- the layers of a decode step on 4-bit weights
// (qllama_model.h): RMSNorm with the residual's addition and an optional Q8_0
// output, the 4-bit weight matrices, and products of a few rows with them.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <new>
#include <type_traits>

#include "../../include/qllama_model.h"
#include "ql_device.cuh"
#include "ql_internal.h"

namespace {

#define QLN_CUDA(call, what)                                                                   \
  do {                                                                                         \
    cudaError_t e_ = (call);                                                                   \
    if (e_ != cudaSuccess)                                                                     \
      return ql_fail(e_ == cudaErrorMemoryAllocation ? QL_ERR_OOM : QL_ERR_CUDA, "%s: %s",    \
                     what, cudaGetErrorString(e_));                                            \
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
  float eps;
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

// Q8_0 block scale of a block whose largest magnitude is `most`; a value v has
// the code round_away(v * inv), within [-limit, limit] once v is cut to
// +-*limit (infinite unless the scale saturates).
__device__ __forceinline__ __half q8_scale(uint32_t most, float& inv, float& limit) {
  limit = INFINITY;
  inv = 0.f;
  if (most >= 0x7f800000u) {
    limit = 0.f;
    return __ushort_as_half(0x7fff);
  }
  float d = __uint_as_float(most) / 127.0f;
  if (d > 65504.0f) {
    d = 65504.0f;
    limit = 127.0f * 65504.0f;
  }
  if (d > 0.f) inv = 1.0f / d;
  return __float2half_rn(d);
}

__device__ __forceinline__ int q8_code(float y, float inv, float limit) {
  if (limit != INFINITY) y = limit == 0.f ? 0.f : fminf(fmaxf(y, -limit), limit);
  return round_away(y * inv);
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
  float inv = 1.0f / sqrtf(ss / static_cast<float>(a.hidden) + a.eps);
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
        static_cast<int8_t*>(a.out)[oo + i] = static_cast<int8_t>(q8_code(y, id, limit));
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
// last go element by element (2000 rows of 4101 bf16 columns: 52.8 us with
// element-wise loads throughout).
constexpr int kNormMax = 16384;  // 512 threads x 32 columns
template <int DT, int WT, int NV, bool LEAD>
__global__ void __launch_bounds__(NV == 1 ? 1024 : 512, NV == 1 ? 1 : 2)
    rms_norm_kernel(const NormArgs a) {
  __shared__ float red[32];
  __shared__ double red_d[32];
  const size_t row = blockIdx.x;
  const size_t oo = row * static_cast<size_t>(a.hidden);
  const int lead = LEAD ? static_cast<int>(oo % 8) : 0;
  ql::griddep_wait();
  ql::griddep_launch_dependents();
  // where x and the residual fill the registers, the weight is left for later
  constexpr bool kEarly = NV * (DT == ql::kF32 ? 2 : 1) < 4;
  Raw8<DT> xr[NV], rr[NV];
  Raw8<WT> wr[NV];
  auto column = [&](int j) { return 8 * static_cast<int>(threadIdx.x + j * blockDim.x) - lead; };
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
  ss = block_sum(ss, red);
  float inv = 1.0f / sqrtf(ss / static_cast<float>(a.hidden) + a.eps);
  if (!plain_square_sum(ss)) {
    // the same for every thread: 64 bits, and s becomes s * inv here
    double sd = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sd += static_cast<double>(s[j][e]) * s[j][e];
    const double id =
        1.0 / sqrt(block_sum(sd, red_d) / a.hidden + static_cast<double>(a.eps));
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
    uint32_t q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = static_cast<uint32_t>(q8_code(y[e], id, limit));
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
// (every kernel here waits for that kernel's end before it touches a tensor).
template <typename... P, typename... A>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                       bool pdl, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// NV: a few rows go over as many threads as they have groups (one round trip,
// the shortest reduction); with two rows or more for every SM, twice as many
// columns a thread (fewer threads wait in a reduction).
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
    return launch_pdl(rms_norm_loop_kernel, dim3(a.rows), dim3(kNormThreads), 0, s, true, a);
  const int groups = (a.hidden + 7) / 8 + lead;
  int nv = groups <= 1024 ? 1 : 4;
  if (nv == 1 && a.rows >= 2 * num_sms && groups >= 256) nv = 2;
  const int threads = ((groups + nv - 1) / nv + 31) / 32 * 32;
  const dim3 grid(a.rows), block(threads);
  auto go = [&](auto dt, auto wt, auto ld) {
    constexpr int DT = decltype(dt)::value, WT = decltype(wt)::value;
    constexpr bool LEAD = decltype(ld)::value;
    if (nv == 1) return launch_pdl(rms_norm_kernel<DT, WT, 1, LEAD>, grid, block, 0, s, true, a);
    if (nv == 2) return launch_pdl(rms_norm_kernel<DT, WT, 2, LEAD>, grid, block, 0, s, true, a);
    return launch_pdl(rms_norm_kernel<DT, WT, 4, LEAD>, grid, block, 0, s, true, a);
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
  // Written since the last product: the next one starts only when all work
  // queued before it is done, and may not read the weights ahead.
  mutable bool fresh = true;
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

template <int FROM>
int launch_pack(ql_q4* w, PackArgs a) {
  a.w = view_of(w);
  w->fresh = true;
  const size_t blocks = (q4_words(w) + 255) / 256;
  q4_pack_kernel<FROM><<<static_cast<unsigned>(blocks), 256, 0, w->ctx->stream>>>(a);
  QLN_CUDA(cudaGetLastError(), "launch the 4-bit layout");
  return QL_OK;
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
// The weights' bytes (0.53-0.56 of them per weight) are the cost of a few rows, so
// they stream straight from HBM into the registers of the lanes that multiply them,
// 16 bytes a lane, with the next ones in flight while one set is multiplied.
// A warp owns MT tiles of 16 weight rows and every 8th chunk of 64 columns; the
// weights are the A operand (16 rows of W), x the B operand (8 columns), so one
// row of x costs as much as eight.  Codes turn into f16 / bf16 exactly (a nibble
// in the mantissa of 1024 or 128, less an offset), or into int8 (a two's-complement
// nibble in the high half of a byte: 16 times its value).  Blocks of 32 sum on the
// tensor cores in f32 (int32 for Q8_0: exact), are scaled in f32 and added to f32
// sums.  f32 rows: three bf16 parts of 8 significand bits each carry a value's 24
// exactly; the parts are three columns of B, whose sums are added at the end.
// The split of the columns over the warps and every order of additions are the
// same for all MT, NT and row counts, so a row's bits depend only on it and W.
constexpr int kLinWarps = 8;
constexpr int kLinThreads = 32 * kLinWarps;

// D = A B (no addend)
template <bool BF>
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
  if constexpr (BF) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  }
}

__device__ __forceinline__ uint4 ld_weights(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// (a & b) ^ c
__device__ __forceinline__ uint32_t and_xor(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// A word's eight values as four pairs in x's order, exactly.
template <bool BF>
__device__ __forceinline__ void unpack_word(uint32_t w, uint32_t (&p)[4]) {
  if constexpr (BF) {
    const uint32_t in[4] = {w, w >> 8, w >> 4, w >> 12};
    const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308),
                                                  __ushort_as_bfloat16(0x4308));  // 136
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t h = and_xor(in[i], 0x000f000fu, 0x43084308u);  // 128 + (value + 8)
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

template <int IN, int NT, int MT, int G>
struct LinCfg {
  static constexpr bool kQ8 = IN == ql::kQ8_0;
  static constexpr bool kBF = IN == ql::kBF16 || IN == ql::kF32;
  static constexpr int kParts = IN == ql::kF32 ? 3 : 1;
  static constexpr int kRows = 8 * NT / kParts;  // rows of x in one pass
  static constexpr int kU = MT >= 4 ? 1 : 4 / MT;  // chunks of one set
  static constexpr int kXWords = kQ8 ? 2 : 4;      // words of a block of 32 in a lane
  static constexpr int kPitch = 16 * MT + 4;
  static constexpr int kSmem = kLinWarps * 8 * NT * kPitch * 4;
};

// One set of loads: U chunks of MT tiles, with x.
template <int IN, int NT, int MT, int G>
struct LinSet {
  using C = LinCfg<IN, NT, MT, G>;
  uint4 w[C::kU][MT];
  uint2 s[C::kU][MT];  // f16: rows g, g + 8 of block j in .x / .y; G >= 64: .x alone
  uint32_t x[C::kU][NT][2][C::kXWords];
  float sx[C::kQ8 ? C::kU : 1][C::kQ8 ? NT : 1][2][2];  // [block][column 2t, 2t + 1]
};

template <int IN, int NT, int MT, int G>
__global__ void __launch_bounds__(kLinThreads) linear_q4_kernel(const LinearArgs a) {
  using C = LinCfg<IN, NT, MT, G>;
  extern __shared__ float red[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tile0 = blockIdx.x * MT;
  const int r0 = blockIdx.y * C::kRows;
  const int rows = min(a.rows - r0, C::kRows);
  const int chunks = a.w.chunks, steps = (chunks + kLinWarps - 1) / kLinWarps;

  using Set = LinSet<IN, NT, MT, G>;
  auto load_w = [&](Set& z, int step) {
#pragma unroll
    for (int u = 0; u < C::kU; ++u) {
      const int chunk = (step + u) * kLinWarps + warp;
      const bool ok = chunk < chunks;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const size_t tile = min(tile0 + m, a.w.tiles - 1);  // past the end: not stored
        z.w[u][m] = make_uint4(0, 0, 0, 0);
        z.s[u][m] = make_uint2(0, 0);
        if (ok) {
          z.w[u][m] = ld_weights(a.w.codes + ((tile * chunks + chunk) * 32 + lane) * 4);
          const __half* sp = a.w.scales + scale_at(G, chunks, tile, chunk, g, 0, 0);
          if constexpr (G == 32) z.s[u][m] = __ldg(reinterpret_cast<const uint2*>(sp));
          else z.s[u][m].x = __ldg(reinterpret_cast<const uint32_t*>(sp));
        }
      }
    }
  };
  // this lane's column of each B tile: a row of x (and a part of it)
  const char* xrow[NT];
  bool live[NT];
  constexpr int kBytes = IN == ql::kF32 ? 4 : C::kQ8 ? 1 : 2;
  const bool vec = (reinterpret_cast<uintptr_t>(a.x) | static_cast<uintptr_t>(a.x_stride * kBytes)) %
                       (C::kQ8 ? 8 : 16) == 0;
  uint32_t m1[NT], m2[NT];  // f32: the bits that parts 1 and 2 take off first
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = 8 * n + g;
    const int r = col / C::kParts, part = col % C::kParts;
    live[n] = r < rows;
    xrow[n] = static_cast<const char*>(a.x) +
              static_cast<size_t>(r0 + (live[n] ? r : 0)) * a.x_stride * kBytes;
    m1[n] = part >= 1 ? 0xffff0000u : 0u;
    m2[n] = part == 2 ? 0xffff0000u : 0u;
  }
  auto load_x = [&](Set& z, int step) {
#pragma unroll
    for (int u = 0; u < C::kU; ++u) {
      const int chunk = (step + u) * kLinWarps + warp;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = 64 * chunk + 32 * j;
        const bool ok = k < a.w.k;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t(&o)[C::kXWords] = z.x[u][n][j];
#pragma unroll
          for (int i = 0; i < C::kXWords; ++i) o[i] = 0;
          if (ok && live[n]) {
            const char* p = xrow[n] + static_cast<size_t>(k + 8 * t) * kBytes;
            if constexpr (C::kQ8) {
              if (vec) {
                const uint2 v = *reinterpret_cast<const uint2*>(p);
                o[0] = v.x;
                o[1] = v.y;
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  o[e / 4] |= static_cast<uint32_t>(reinterpret_cast<const uint8_t*>(p)[e])
                              << (8 * (e % 4));
              }
            } else if constexpr (IN == ql::kF32) {
              uint32_t f[8];
              if (vec) {
                const uint4 v = reinterpret_cast<const uint4*>(p)[0];
                const uint4 q = reinterpret_cast<const uint4*>(p)[1];
                f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
                f[4] = q.x; f[5] = q.y; f[6] = q.z; f[7] = q.w;
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = reinterpret_cast<const uint32_t*>(p)[e];
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                float v = __uint_as_float(f[e]);
                v -= __uint_as_float(__float_as_uint(v) & m1[n]);
                v -= __uint_as_float(__float_as_uint(v) & m2[n]);
                f[e] = __float_as_uint(v);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) o[i] = __byte_perm(f[2 * i], f[2 * i + 1], 0x7632);
            } else {
              if (vec) {
                const uint4 v = *reinterpret_cast<const uint4*>(p);
                o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  o[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[e])
                              << (16 * (e % 2));
              }
            }
          }
          if constexpr (C::kQ8) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int r = 8 * n + 2 * t + c;
              z.sx[u][n][j][c] = 0.f;
              if (ok && r < rows)  // 1/16: the codes are 16 times their values
                z.sx[u][n][j][c] =
                    0.0625f * __half2float(a.x_scale[static_cast<size_t>(r0 + r) * (a.w.k / 32) +
                                                     k / 32]);
            }
          }
        }
      }
    }
  };

  float acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.f;

  auto multiply = [&](const Set& z) {
#pragma unroll
    for (int u = 0; u < C::kU; ++u) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint32_t w[4] = {z.w[u][m].x, z.w[u][m].y, z.w[u][m].z, z.w[u][m].w};
        if constexpr (C::kQ8) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t sw = G == 32 && j == 1 ? z.s[u][m].y : z.s[u][m].x;
            const float2 s = __half22float2(*reinterpret_cast<const __half2*>(&sw));
            const uint4 A = make_uint4((w[2 * j] << 4) & 0xf0f0f0f0u, (w[2 * j + 1] << 4) & 0xf0f0f0f0u,
                                       w[2 * j] & 0xf0f0f0f0u, w[2 * j + 1] & 0xf0f0f0f0u);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              // sums start at the bits of 1.5 * 2^23: below 2^22 they are the
              // mantissa of a float, and a subtraction converts them
              int d[4] = {0x4b400000, 0x4b400000, 0x4b400000, 0x4b400000};
              ql::mma16832_s8(d, A, __byte_perm(z.x[u][n][j][0], 0, 0x3120),
                              __byte_perm(z.x[u][n][j][1], 0, 0x3120));
#pragma unroll
              for (int i = 0; i < 4; ++i)
                acc[m][n][i] = fmaf(__int_as_float(d[i]) - 12582912.0f,
                                    (i < 2 ? s.x : s.y) * z.sx[u][n][j][i & 1], acc[m][n][i]);
            }
          }
        } else {
          uint32_t lo[2][4], hi[2][4];  // rows g and g + 8 of both blocks
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            unpack_word<C::kBF>(w[2 * j], lo[j]);
            unpack_word<C::kBF>(w[2 * j + 1], hi[j]);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float d[4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t A0[4] = {lo[j][0], hi[j][0], lo[j][1], hi[j][1]};
              const uint32_t A1[4] = {lo[j][2], hi[j][2], lo[j][3], hi[j][3]};
              if (G == 32 || j == 0)
                mma16816_first<C::kBF>(d, A0, z.x[u][n][j][0], z.x[u][n][j][1]);
              else
                ql::mma16816<C::kBF>(d, A0, z.x[u][n][j][0], z.x[u][n][j][1]);
              ql::mma16816<C::kBF>(d, A1, z.x[u][n][j][2], z.x[u][n][j][3]);
              if (G == 32 || j == 1) {
                const uint32_t sw = G == 32 && j == 1 ? z.s[u][m].y : z.s[u][m].x;
                const float2 s = __half22float2(*reinterpret_cast<const __half2*>(&sw));
                acc[m][n][0] = fmaf(d[0], s.x, acc[m][n][0]);
                acc[m][n][1] = fmaf(d[1], s.x, acc[m][n][1]);
                acc[m][n][2] = fmaf(d[2], s.y, acc[m][n][2]);
                acc[m][n][3] = fmaf(d[3], s.y, acc[m][n][3]);
              }
            }
          }
        }
      }
    }
  };

  // The first weights do not depend on the kernel before this one (a product
  // after a write of the weights is launched without the overlap).
  Set z0, z1;
  load_w(z0, 0);
  ql::griddep_wait();
  ql::griddep_launch_dependents();
  load_x(z0, 0);
  for (int step = 0; step < steps; step += 2 * C::kU) {
    if (step + C::kU < steps) {
      load_w(z1, step + C::kU);
      load_x(z1, step + C::kU);
    }
    multiply(z0);
    if (step + C::kU >= steps) break;
    if (step + 2 * C::kU < steps) {
      load_w(z0, step + 2 * C::kU);
      load_x(z0, step + 2 * C::kU);
    }
    multiply(z1);
  }

  // join the warps: red[warp][column][row]
  float* mine = red + static_cast<size_t>(warp) * 8 * NT * C::kPitch;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        mine[(8 * n + 2 * t + (i & 1)) * C::kPitch + 16 * m + g + 8 * (i >> 1)] = acc[m][n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * MT * rows; i += kLinThreads) {
    const int row = i % (16 * MT), r = i / (16 * MT);
    const int n = tile0 * 16 + row;
    if (n >= a.w.n) continue;
    float y = 0.f;
#pragma unroll
    for (int p = C::kParts - 1; p >= 0; --p) {  // the small parts first
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kLinWarps; ++w)
        v += red[(static_cast<size_t>(w) * 8 * NT + r * C::kParts + p) * C::kPitch + row];
      y += v;
    }
    ql::store_elem(a.y, static_cast<size_t>(r0 + r) * a.y_stride + n, a.out_dtype, y);
  }
}

template <int IN, int NT, int MT, int G>
cudaError_t launch_linear_as(const LinearArgs& a, bool pdl, cudaStream_t s) {
  using C = LinCfg<IN, NT, MT, G>;
  const int kern_smem = C::kSmem;
  if constexpr (C::kSmem > 48 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(linear_q4_kernel<IN, NT, MT, G>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
  }
  for (int r = 0; r < a.rows; r += 65535 * C::kRows) {  // grid.y holds 65535 passes
    LinearArgs b = a;
    b.rows = std::min(a.rows - r, 65535 * C::kRows);
    const size_t xb = type_bytes(a.in_dtype), yb = type_bytes(a.out_dtype);
    b.x = static_cast<const char*>(a.x) + static_cast<size_t>(r) * a.x_stride * xb;
    b.x_scale = a.x_scale ? a.x_scale + static_cast<size_t>(r) * (a.w.k / 32) : nullptr;
    b.y = static_cast<char*>(a.y) + static_cast<size_t>(r) * a.y_stride * yb;
    const dim3 grid((a.w.tiles + MT - 1) / MT, (b.rows + C::kRows - 1) / C::kRows);
    const cudaError_t e =
        launch_pdl(linear_q4_kernel<IN, NT, MT, G>, grid, dim3(kLinThreads), kern_smem, s, pdl, b);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <int IN, int G>
cudaError_t launch_linear_in(const LinearArgs& a, bool pdl, cudaStream_t s) {
  const int columns = a.rows * (IN == QL_F32 ? 3 : 1);
  int mt = columns <= 8 ? 1 : columns <= 16 ? 2 : 4;
  if (const char* e = getenv("QLMT")) mt = atoi(e);
  if (columns <= 8) return mt == 1 ? launch_linear_as<IN, 1, 1, G>(a, pdl, s) : launch_linear_as<IN, 1, 2, G>(a, pdl, s);
  if (columns <= 16) return mt == 1 ? launch_linear_as<IN, 2, 1, G>(a, pdl, s) : mt == 2 ? launch_linear_as<IN, 2, 2, G>(a, pdl, s) : launch_linear_as<IN, 2, 4, G>(a, pdl, s);
  return mt == 2 ? launch_linear_as<IN, 4, 2, G>(a, pdl, s) : launch_linear_as<IN, 4, 4, G>(a, pdl, s);
}

cudaError_t launch_linear(const LinearArgs& a, bool pdl, cudaStream_t s) {
  auto by_group = [&](auto in) {
    constexpr int IN = decltype(in)::value;
    if (a.w.group == 32) return launch_linear_in<IN, 32>(a, pdl, s);
    if (a.w.group == 64) return launch_linear_in<IN, 64>(a, pdl, s);
    return launch_linear_in<IN, 128>(a, pdl, s);
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
  if (out_features > (1 << 30) || in_features > (1 << 30))
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
    return ql_fail(e == cudaErrorMemoryAllocation ? QL_ERR_OOM : QL_ERR_CUDA,
                   "allocate a 4-bit weight: %s", cudaGetErrorString(e));
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
  QLN_CUDA(launch_linear(a, !w->fresh, c->stream), "launch the 4-bit product");
  w->fresh = false;
  return QL_OK;
}

}  // extern "C"
