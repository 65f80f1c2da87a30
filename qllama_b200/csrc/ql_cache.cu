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

}  // namespace

// ---------------------------------------------------------------- append --
// One warp per row: token r's query heads, then its KV heads.
__global__ void __launch_bounds__(128) ragged_append_kernel(const __grid_constant__ RaggedAppendArgs a) {
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const CacheView& c = a.cache;
  const int heads = a.hq + c.hkv, hd = c.hd;
  const int64_t r64 = warp / heads;
  if (r64 >= a.rows.first[a.batch]) return;
  const int r = static_cast<int>(r64), h = static_cast<int>(warp - r64 * heads);
  const int b = ragged_seq(a.rows, a.batch, r);
  const int pos = a.rows.start[b] + r - a.rows.first[b];
  const double2* rope = a.rope + static_cast<size_t>(pos) * (hd / 2);
  if (h < a.hq) {
    const size_t in = static_cast<size_t>(r) * a.q_stride + static_cast<size_t>(h) * hd;
    const size_t out = (static_cast<size_t>(r) * a.hq + h) * hd;
    for (int p = lane; p < hd / 2; p += 32) {
      float y0, y1;
      rope_pair(load_elem(a.q, in + 2 * p, a.in_dtype), load_elem(a.q, in + 2 * p + 1, a.in_dtype),
                rope[p], y0, y1);
      store_elem(a.q_out, out + 2 * p, a.q_out_dtype, y0);
      store_elem(a.q_out, out + 2 * p + 1, a.q_out_dtype, y1);
    }
    return;
  }
  const int kvh = h - a.hq;
  bool ok;
  const int64_t dst = cache_row(c, a.rows.seq[b], pos, kvh, a.status, ok);
  if (!ok) return;
  append_row(a.k, a.v, a.in_dtype, static_cast<size_t>(r) * a.k_stride + static_cast<size_t>(kvh) * hd,
             static_cast<size_t>(r) * a.v_stride + static_cast<size_t>(kvh) * hd, rope, c, dst, lane);
}

cudaError_t launch_ragged_append(const RaggedAppendArgs& a, cudaStream_t s) {
  const int64_t warps = static_cast<int64_t>(a.rows.first[a.batch]) * (a.hq + a.cache.hkv);
  if (warps == 0) return cudaSuccess;
  ragged_append_kernel<<<static_cast<unsigned>((warps + 3) / 4), 128, 0, s>>>(a);
  return cudaGetLastError();
}

// ------------------------------------------------------------------ read --
// One warp per (token, KV head).
__global__ void __launch_bounds__(128) ragged_read_kernel(const __grid_constant__ RaggedReadArgs a) {
  const int64_t warp = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const CacheView& c = a.cache;
  const int64_t r64 = warp / c.hkv;
  if (r64 >= a.rows.first[a.batch]) return;
  const int r = static_cast<int>(r64), h = static_cast<int>(warp - r64 * c.hkv);
  const int b = ragged_seq(a.rows, a.batch, r);
  bool ok;
  const int64_t row = cache_row(c, a.rows.seq[b], a.rows.start[b] + r - a.rows.first[b], h,
                                a.status, ok);
  const size_t o = static_cast<size_t>(warp) * c.hd;
  for (int d = lane; d < c.hd; d += 32) {
    store_elem(a.k_out, o + d, a.out_dtype, ok ? cache_value(c, false, row, d) : 0.f);
    store_elem(a.v_out, o + d, a.out_dtype, ok ? cache_value(c, true, row, d) : 0.f);
  }
}

cudaError_t launch_ragged_read(const RaggedReadArgs& a, cudaStream_t s) {
  const int64_t warps = static_cast<int64_t>(a.rows.first[a.batch]) * a.cache.hkv;
  if (warps == 0) return cudaSuccess;
  ragged_read_kernel<<<static_cast<unsigned>((warps + 3) / 4), 128, 0, s>>>(a);
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
// bf16.  A channel that holds a NaN gets NaN bounds.
__global__ void __launch_bounds__(128) bounds_kernel(const __grid_constant__ BoundsArgs a) {
  const CacheView& c = a.cache;
  const int kvh = blockIdx.y;
  const int b = ragged_seq(a.blocks, a.batch, blockIdx.x);
  const int block = a.blocks.start[b] + static_cast<int>(blockIdx.x) - a.blocks.first[b];
  bool ok;
  const int64_t row = cache_row(c, a.blocks.seq[b], block * kTile, kvh, a.status, ok);
  if (!ok) return;
  const int page = static_cast<int>(row / c.page / c.hkv);
  uint16_t* out = a.bounds + bounds_row(c, page, block, kvh);
  for (int d = threadIdx.x; d < c.hd; d += blockDim.x) {
    float lo = CUDART_INF_F, hi = -CUDART_INF_F;
    bool nan = false;
    for (int i = 0; i < kTile; ++i) {
      const float x = cache_value(c, false, row + i, d);
      nan |= x != x;
      lo = fminf(lo, x);
      hi = fmaxf(hi, x);
    }
    if (nan) lo = hi = CUDART_NAN_F;
    const bool half = c.dtype == kF16;
    out[d] = static_cast<uint16_t>(half ? pack2<false>(lo, lo) : pack2<true>(lo, lo));
    out[c.hd + d] = static_cast<uint16_t>(half ? pack2<false>(hi, hi) : pack2<true>(hi, hi));
  }
}

cudaError_t launch_bounds(const BoundsArgs& a, cudaStream_t s) {
  const int n = a.blocks.first[a.batch];
  if (n == 0) return cudaSuccess;
  bounds_kernel<<<dim3(n, a.cache.hkv), 128, 0, s>>>(a);
  return cudaGetLastError();
}

namespace {

constexpr int kChooseThreads = 256;
constexpr int kChooseBlocks = 64;  // scored by one CTA
constexpr int kBins = 2048;

// Eight consecutive values of a bounds row.
__device__ __forceinline__ void load_bounds(const uint16_t* p, bool half, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
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

__device__ __forceinline__ double block_extreme(double v, bool largest, double* red) {
  for (int o = 16; o > 0; o >>= 1) {
    const double w = __shfl_xor_sync(0xffffffffu, v, o);
    v = largest ? fmax(v, w) : fmin(v, w);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int i = 0; i < kChooseThreads / 32; ++i) v = largest ? fmax(v, red[i]) : fmin(v, red[i]);
  return v;
}

}  // namespace

// Scores and choice in one launch.  The CTAs of a (token, KV head) score kChooseBlocks blocks
// each; the last to arrive chooses.
//
// Scores: the group's queries enter by the sums of their positive and of their negative parts,
// because sum_h max(q_h lo, q_h hi) = (sum_h max(q_h, 0)) hi + (sum_h min(q_h, 0)) lo while
// lo <= hi: two products a channel whatever the group.  In f64, so that only equal blocks tie.
// Eight lanes a block (HD 64 or 128), else (HD 0) a warp.  Bound by the bounds' bytes.
//
// Choice: a histogram over the range of the scores puts the border into one of kBins bins;
// those above it are in, and the few in it are ranked among themselves by (score, block).
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
  const int chunks = (hi_block + kChooseBlocks - 1) / kChooseBlocks;
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
    const int block0 = blockIdx.x * kChooseBlocks, end = min(block0 + kChooseBlocks, hi_block);
    if constexpr (HD != 0) {
      constexpr int kPer = HD / 64;  // lane `sub` of eight: dims 64 j + 8 sub .. + 7
      const int sub = lane & 7;
      double up[kPer][8], down[kPer][8];
#pragma unroll
      for (int j = 0; j < kPer; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) up[j][k] = down[j][k] = 0.0;
      for (int h = 0; h < a.group; ++h)
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          float x[4], y[4];
          const size_t at = q0 + static_cast<size_t>(h) * HD + 64 * j + 8 * sub;
          load_vec<4>(a.q, at, a.in_dtype, a.q_vec != 0, x);
          load_vec<4>(a.q, at + 4, a.in_dtype, a.q_vec != 0, y);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            add_parts(x[k], up[j][k], down[j][k]);
            add_parts(y[k], up[j][k + 4], down[j][k + 4]);
          }
        }
      for (int base = block0 + 4 * warp; base < end; base += kChooseThreads / 8) {
        const int block = base + (lane >> 3);
        const uint16_t* p = block < end && block >= lo_block ? bounds_of(block) : nullptr;
        double s = 0.0;
        if (p) {
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            float lo[8], hi[8];
            load_bounds(p + 64 * j + 8 * sub, half, lo);
            load_bounds(p + HD + 64 * j + 8 * sub, half, hi);
#pragma unroll
            for (int k = 0; k < 8; ++k) s += up[j][k] * hi[k] + down[j][k] * lo[k];
          }
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (s != s) s = CUDART_INF;  // a NaN counts as the largest score
        if (p && sub == 0) score[block] = s;
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
        if (s != s) s = CUDART_INF;
        if (lane == 0) score[block] = s;
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
  __shared__ double red[kChooseThreads / 32];
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
    for (int j = lo_block + threadIdx.x; j < hi_block; j += kChooseThreads) {
      const double s = __ldcg(score + j);
      if (fits) dyn[j] = s;
      if (fabs(s) < CUDART_INF) {
        least = fmin(least, s);
        most = fmax(most, s);
      }
    }
    least = block_extreme(least, false, red);
    most = block_extreme(most, true, red);
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
    int32_t* out = sel + done + before - n;
    for (; w; w &= w - 1) *out++ = 32 * (w0 + lane) + __ffs(w) - 1;
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
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.max_blocks + kChooseBlocks - 1) / kChooseBlocks, a.cache.hkv, jobs);
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
