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

// One warp per (token, KV head, block).  The group's queries enter by the sums of their
// positive and of their negative parts, because sum_h max(q_h lo, q_h hi) = (sum_h max(q_h, 0)) hi
// + (sum_h min(q_h, 0)) lo while lo <= hi.  In f64, so that only equal blocks tie.
__global__ void __launch_bounds__(128) score_kernel(const __grid_constant__ SelectArgs a) {
  const CacheView& c = a.cache;
  const int lane = threadIdx.x & 31;
  const int block = blockIdx.x * 4 + (threadIdx.x >> 5), kvh = blockIdx.y, job = blockIdx.z;
  const int b = job / a.new_len, qpos = a.seqs.start[b] + job % a.new_len;
  if (block >= qpos / kTile) return;
  bool ok;
  const int64_t row = cache_row(c, a.seqs.seq[b], block * kTile, kvh, a.status, ok);
  double s = 0.0;
  if (ok) {
    const int page = static_cast<int>(row / c.page / c.hkv);
    const uint16_t* lo = a.bounds + bounds_row(c, page, block, kvh);
    const int bt = c.dtype == kF16 ? kF16 : kBF16;
    for (int d = lane; d < c.hd; d += 32) {
      double up = 0.0, down = 0.0;
      for (int h = 0; h < a.group; ++h) {
        const double x = load_elem(
            a.q, (static_cast<size_t>(job) * a.hq + kvh * a.group + h) * c.hd + d, a.in_dtype);
        if (x > 0.0) up += x;
        else down += x;  // a NaN lands here
      }
      s += up * load_elem(lo, c.hd + d, bt) + down * load_elem(lo, d, bt);
    }
  }
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (s != s) s = CUDART_INF;  // a NaN counts as the largest score
  if (lane == 0) a.score[(static_cast<size_t>(job) * c.hkv + kvh) * a.max_blocks + block] = s;
}

// One CTA per (token, KV head): each block's rank among the scores.
__global__ void __launch_bounds__(256) select_kernel(const __grid_constant__ SelectArgs a) {
  const CacheView& c = a.cache;
  const int kvh = blockIdx.x, job = blockIdx.y;
  const int b = job / a.new_len, qpos = a.seqs.start[b] + job % a.new_len;
  const int count = qpos / kTile + 1;
  const size_t pair = static_cast<size_t>(job) * c.hkv + kvh;
  const double* score = a.score + pair * a.max_blocks;
  int32_t* sel = a.sel + pair * a.take;
  extern __shared__ uint8_t chosen[];  // [count]
  auto forced = [&](int j) { return j < a.first || j >= count - a.last; };
  const int free = a.take - min(a.first, count) - a.last;
  for (int j = threadIdx.x; j < count; j += blockDim.x) {
    bool in = count <= a.take || forced(j);
    if (!in) {
      const double s = score[j];
      int rank = 0;
      for (int i = a.first; i < count - a.last; ++i)
        rank += score[i] > s || (score[i] == s && i < j);
      in = rank < free;
    }
    chosen[j] = in;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int j = 0; j < count; ++j)
      if (chosen[j]) sel[n++] = j;
    for (; n < a.take; ++n) sel[n] = -1;
  }
}

cudaError_t launch_select(const SelectArgs& a, cudaStream_t s) {
  const int jobs = a.batch * a.new_len;
  score_kernel<<<dim3((a.max_blocks + 3) / 4, a.cache.hkv, jobs), 128, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  select_kernel<<<dim3(a.cache.hkv, jobs), 256, a.max_blocks, s>>>(a);
  return cudaGetLastError();
}

}  // namespace ql
