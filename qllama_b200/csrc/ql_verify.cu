// ql_verify.cu -- verification of drafted tokens (qllama_model.h): speculative
// sampling's acceptance and the draw of the next token, beside ql_sample.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>

#include "../../include/qllama_model.h"
#include "ql_device.cuh"
#include "ql_internal.h"

namespace {

#define QLV_CUDA(call, what)                                                      \
  do {                                                                            \
    cudaError_t e_ = (call);                                                      \
    if (e_ != cudaSuccess)                                                        \
      return ql_fail(QL_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e_));        \
  } while (0)

struct VerifyArgs {
  const void* target;
  const void* draft;
  const int32_t* ids;
  const int32_t* n_draft;
  const double* uniforms;
  int32_t* tokens;
  int32_t* accepted;
  uint32_t* status;
  int64_t target_stride, draft_stride;
  int drafts, vocab, dtype, probs;
  double inv_t;  // 1 / temperature; 0: greedy
};

// One cluster of CTAs per sequence, each CTA with its share of every row.
//   1. f32 (maximum, sum of exponentials) of all of the sequence's rows at once --
//      the one pass over the logits, bound by their bytes -- joined over the cluster
//      through distributed shared memory.  (Greedy: largest logit and its id.)
//   2. Every draft is decided from its two logits and those sums.  A decision whose
//      two sides are within 2^-14 of each other, far more than the f32 sums' error, is
//      taken again from f64 sums of its rows.
//   3. The rows at the first rejection (or the last row) are summed again in f64: the
//      draw compares running sums over the whole vocabulary with a threshold, where an
//      error of 1e-7 would change one token in some thousands.  The CTA, the warp and
//      the lane where the running sum of the draw passes the threshold are found in
//      turn.
// All CTAs compute the same decisions from the same numbers, so the cluster's
// barriers are met by all.  Nothing is kept outside shared memory.
constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyRows = 2 * QL_VERIFY_MAX_DRAFTS + 1;
constexpr int kMaxCluster = 16;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float2 ld_cluster_f2(const void* p, uint32_t rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(ql::mapa_shared(ql::smem_u32(p), rank))
               : "memory");
  return v;
}
__device__ __forceinline__ double ld_cluster_f64(const void* p, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];"
               : "=d"(v)
               : "r"(ql::mapa_shared(ql::smem_u32(p), rank))
               : "memory");
  return v;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp(d / T) in f64 for d <= 0 by the table method (P. T. P. Tang, 1989):
// d / T = (k + r) ln2 / 32 with |r| <= 1/2, k = 32 e + j; the result is
// 2^e 2^(j/32) exp(r ln2 / 32), the last by five terms of its series (the sixth is
// below 3e-15).  Lane j holds 2^(j/32), read by shuffles: whole warps call this.
struct Exp64 {
  double table, scale, least;
  __device__ explicit Exp64(double inv_t) {
    constexpr double ln2 = 0.693147180559945309417232;
    table = exp2(static_cast<double>(threadIdx.x & 31) / 32.0);
    scale = inv_t * (32.0 / ln2);
    least = -690.0 / inv_t;  // below it the result is taken as 0 (it is under 1e-299)
  }
  __device__ __forceinline__ double operator()(double d) const {
    constexpr double L = 0.693147180559945309417232 / 32.0;
    constexpr double magic = 6755399441055744.0;  // 1.5 * 2^52
    const bool in = d >= least;
    if (!in) d = 0.0;
    const double t = fma(d, scale, magic);
    const int k = __double2loint(t);
    const double r = fma(d, scale, magic - t);
    double p = fma(r, L * L * L * L * L / 120, L * L * L * L / 24);
    p = fma(p, r, L * L * L / 6);
    p = fma(p, r, L * L / 2);
    p = fma(p, r, L);
    p = fma(p, r, 1.0);
    const int hi = __shfl_sync(0xffffffffu, __double2hiint(table), k & 31) + ((k >> 5) << 20);
    const int lo = __shfl_sync(0xffffffffu, __double2loint(table), k & 31);
    return in ? p * __hiloint2double(hi, lo) : 0.0;
  }
};

// A row's 16-byte groups: element e of the row is element (e + shift) of the groups.
template <int DT>
struct Groups {
  static constexpr int kN = DT == ql::kF32 ? 4 : 8;
  const uint4* base;
  int shift, count;
  __device__ Groups(const void* p, size_t at, int vocab) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p) + at * (16 / kN);
    shift = static_cast<int>(a % 16) / (16 / kN);
    base = reinterpret_cast<const uint4*>(a - a % 16);
    count = (vocab + shift + kN - 1) / kN;
  }
  // Elements of group i; those outside the row are `fill` (their memory is not read).
  __device__ __forceinline__ void load(int i, int vocab, float fill, float (&x)[kN]) const {
    const int e0 = i * kN - shift;
    if (e0 >= 0 && e0 + kN <= vocab) {
      const uint4 v = base[i];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        if constexpr (DT == ql::kF32) x[e] = __uint_as_float(w[e]);
        else {
          const uint16_t h = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
          if constexpr (DT == ql::kF16) x[e] = __half2float(__ushort_as_half(h));
          else x[e] = __uint_as_float(static_cast<uint32_t>(h) << 16);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < kN; ++e)
        x[e] = e0 + e >= 0 && e0 + e < vocab ? ql::load_elem(base, static_cast<size_t>(i) * kN + e, DT)
                                             : fill;
    }
  }
};

// A row as a distribution: weight(i) / z.
struct Row {
  size_t at;
  float m;
  double z;
};

template <int DT>
__global__ void __launch_bounds__(kVerifyThreads, 1) verify_kernel(const VerifyArgs a) {
  __shared__ float2 part[kVerifyRows][kVerifyWarps];  // a row's (m, s) or (best, id) by warp
  __shared__ float2 mine[kVerifyRows];                // of this CTA
  __shared__ float2 row_stat[kVerifyRows];            // of the cluster
  __shared__ double sums[2][kVerifyWarps];
  __shared__ double share[2][2];  // this CTA's sums, for the cluster (two turns)
  __shared__ int pos_s, exact_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = a.vocab;
  const int rank = static_cast<int>(cluster_rank()), ctas = static_cast<int>(cluster_size());
  const int b = blockIdx.x / ctas;
  ql::griddep_wait();
  ql::griddep_launch_dependents();
  const int n = a.n_draft ? min(max(a.n_draft[b], 0), a.drafts) : a.drafts;
  const int32_t* ids = a.ids + static_cast<size_t>(b) * a.drafts;
  const double* u = a.uniforms + static_cast<size_t>(b) * (a.drafts + 1);
  const bool greedy = a.inv_t == 0, stats = !a.probs;
  const bool has_q = a.draft != nullptr && !greedy;
  auto target_at = [&](int i) {
    return (static_cast<size_t>(b) * (a.drafts + 1) + i) * static_cast<size_t>(a.target_stride);
  };
  auto draft_at = [&](int i) {
    return (static_cast<size_t>(b) * a.drafts + i) * static_cast<size_t>(a.draft_stride);
  };
  // ---- 1. rows 0 .. n: the target's, n + 1 .. 2n: the draft's
  const int nrows = stats ? n + 1 + (has_q ? n : 0) : 0;
  const float c = static_cast<float>(fmin(a.inv_t * 1.4426950408889634, 3e38));
  for (int i = tid; i < nrows * kVerifyWarps; i += kVerifyThreads)
    part[i / kVerifyWarps][i % kVerifyWarps] =
        greedy ? make_float2(-INFINITY, __int_as_float(INT_MAX)) : make_float2(-INFINITY, 0.f);
  __syncthreads();
  if (stats) {
    using G = Groups<DT>;
    constexpr int kLoads = 8;  // groups of a lane in flight
    // items: pieces of 32 * kLoads groups of this CTA's share of a row
    const int most = (V + 2 * G::kN - 2) / G::kN;
    const int span = (most + ctas - 1) / ctas;
    const int pieces = (span + 32 * kLoads - 1) / (32 * kLoads);
    const long long items = static_cast<long long>(pieces) * nrows;
    long long it = items * warp / kVerifyWarps;
    const long long end = items * (warp + 1) / kVerifyWarps;
    int row = static_cast<int>(it / pieces), piece = static_cast<int>(it % pieces);
    while (it < end) {
      const G g(row <= n ? a.target : a.draft, row <= n ? target_at(row) : draft_at(row - n - 1), V);
      const int stop = min(g.count, (rank + 1) * span);
      float m = -INFINITY, s = 0.f;
      int best = INT_MAX, bad = 0;
      for (; it < end && piece < pieces; ++it, ++piece) {
        const int i0 = rank * span + piece * 32 * kLoads + lane;
        float x[kLoads][G::kN];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          if (i0 + 32 * j < stop) {
            g.load(i0 + 32 * j, V, -INFINITY, x[j]);
          } else {
#pragma unroll
            for (int e = 0; e < G::kN; ++e) x[j][e] = -INFINITY;
          }
        }
        if (greedy) {
#pragma unroll
          for (int j = 0; j < kLoads; ++j)
#pragma unroll
            for (int e = 0; e < G::kN; ++e) {  // ascending ids: the first of equals stays
              bad |= !(x[j][e] < INFINITY);
              if (x[j][e] > m) {
                m = x[j][e];
                best = (i0 + 32 * j) * G::kN - g.shift + e;
              }
            }
        } else {
          float top = m;
#pragma unroll
          for (int j = 0; j < kLoads; ++j)
#pragma unroll
            for (int e = 0; e < G::kN; ++e) top = fmaxf(top, x[j][e]);
          if (top == -INFINITY) {  // nothing yet, unless a NaN hides among the -inf
#pragma unroll
            for (int j = 0; j < kLoads; ++j)
#pragma unroll
              for (int e = 0; e < G::kN; ++e) bad |= x[j][e] != x[j][e];
          } else {
            s *= m == -INFINITY ? 0.f : exp2_fast((m - top) * c);
            m = top;
            float add = 0.f;
#pragma unroll
            for (int j = 0; j < kLoads; ++j)
#pragma unroll
              for (int e = 0; e < G::kN; ++e) add += exp2_fast((x[j][e] - top) * c);
            s += add;
          }
        }
      }
      // this warp's part of the row
      if (greedy) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
          const int b2 = __shfl_xor_sync(0xffffffffu, best, o);
          if (m2 > m || (m2 == m && b2 < best)) {
            m = m2;
            best = b2;
          }
        }
        if (__any_sync(0xffffffffu, bad)) m = NAN;
        if (lane == 0) part[row][warp] = make_float2(m, __int_as_float(best));
      } else {
        float top = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        s = m == -INFINITY ? 0.f : s * exp2_fast((m - top) * c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (__any_sync(0xffffffffu, bad)) s = NAN;
        if (lane == 0) part[row][warp] = make_float2(top, s);
      }
      ++row;
      piece = 0;
    }
    __syncthreads();
    // (m, s) or (best, id) of the parts that the lanes of a warp hold
    auto join = [&](float2 r) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float2 v = make_float2(__shfl_xor_sync(0xffffffffu, r.x, o),
                                     __shfl_xor_sync(0xffffffffu, r.y, o));
        if (greedy) {  // NaN: the row is bad
          if (r.x != r.x) continue;
          if (v.x != v.x || v.x > r.x ||
              (v.x == r.x && __float_as_int(v.y) < __float_as_int(r.y)))
            r = v;
        } else {
          const float top = fmaxf(r.x, v.x);
          // sums under a maximum of -inf are zeros, or a NaN that marks the row
          const float f = r.x == top ? 1.f : r.x == -INFINITY ? 0.f : exp2_fast((r.x - top) * c);
          const float h = v.x == top ? 1.f : v.x == -INFINITY ? 0.f : exp2_fast((v.x - top) * c);
          r.y = r.y * f + v.y * h;
          r.x = top;
        }
      }
      return r;
    };
    const float2 none =
        greedy ? make_float2(-INFINITY, __int_as_float(INT_MAX)) : make_float2(-INFINITY, 0.f);
    for (int r = warp; r < nrows; r += kVerifyWarps) {
      const float2 v = join(lane < kVerifyWarps ? part[r][lane] : none);
      if (lane == 0) mine[r] = v;
    }
    cluster_sync();
    for (int r = warp; r < nrows; r += kVerifyWarps) {
      const float2 v = join(lane < ctas ? ld_cluster_f2(&mine[r], lane) : none);
      if (lane == 0) row_stat[r] = v;
    }
    __syncthreads();
  }

  // ---- f64 sums over the cluster; lane k of every warp gets CTA k's first sum
  int turn = 0;
  auto warp_total = [&](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto cluster_sums = [&](double& v0, double& v1) -> double {
    v0 = warp_total(v0);
    v1 = warp_total(v1);
    __syncthreads();  // the warps' sums before have been read
    if (lane == 0) {
      sums[0][warp] = v0;
      sums[1][warp] = v1;
    }
    __syncthreads();
    if (warp < 2) {
      const double s = warp_total(lane < kVerifyWarps ? sums[warp][lane] : 0.0);
      if (lane == 0) share[turn][warp] = s;
    }
    cluster_sync();
    const double p0 = lane < ctas ? ld_cluster_f64(&share[turn][0], lane) : 0.0;
    const double p1 = lane < ctas ? ld_cluster_f64(&share[turn][1], lane) : 0.0;
    v0 = warp_total(p0);
    v1 = warp_total(p1);
    turn ^= 1;  // the other pair next: this one is read until the next barrier
    return p0;
  };
  // this CTA's ids, and this warp's of them
  const int lo = static_cast<int>(static_cast<long long>(V) * rank / ctas);
  const int hi = static_cast<int>(static_cast<long long>(V) * (rank + 1) / ctas);
  auto warp_part = [&](int from, int to, int w) {
    return from + static_cast<int>(static_cast<long long>(to - from) * w / kVerifyWarps);
  };
  const Exp64 ex(greedy ? 1.0 : a.inv_t);
  // Weights of a row at four ids of a lane (their loads, and then the steps of four
  // exponentials, in flight together); whole warps.
  auto weights = [&](const void* base, const Row& r, const int (&i)[4], double (&w)[4]) {
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = ql::load_elem(base, r.at + i[e], DT);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] = a.probs ? static_cast<double>(x[e]) : ex(static_cast<double>(x[e]) - r.m);
  };
  // add(ids, of) over this warp's part of [from, to), 128 ids at a time; ids past the
  // part repeat its last, and `of` says how many of the lane's four are inside
  auto each = [&](int from, int to, auto add) {
    const int f = warp_part(from, to, warp), e = warp_part(from, to, warp + 1);
    for (int i0 = f + lane; i0 - lane < e; i0 += 128) {
      const int i[4] = {min(i0, e - 1), min(i0 + 32, e - 1), min(i0 + 64, e - 1),
                        min(i0 + 96, e - 1)};
      add(i, i0 < e ? min(4, (e - i0 + 31) / 32) : 0);
    }
  };
  auto exact_sums = [&](Row& p, Row& q, bool with_q) {
    if (a.probs) {
      p.z = q.z = 1.0;
      return;
    }
    double sp = 0, sq = 0;
    each(lo, hi, [&](const int(&i)[4], int of) {
      double w[4];
      weights(a.target, p, i, w);
#pragma unroll
      for (int e = 0; e < 4; ++e) sp += e < of ? w[e] : 0.0;
      if (with_q) {
        weights(a.draft, q, i, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) sq += e < of ? w[e] : 0.0;
      }
    });
    cluster_sums(sp, sq);
    p.z = sp;
    q.z = sq;
  };

  // ---- 2. the first draft that is not accepted
  // of[i]: 0 accepted, 1 rejected, 2 too close for the f32 sums, 3 cannot be decided
  auto usable = [&](float2 st) { return st.y > 0.f && st.y < INFINITY && st.x > -INFINITY; };
  auto decide = [&](int i, double zp, double zq, bool exact) {
    const int x = ids[i];
    if (x < 0 || x >= V) return 3;
    if (greedy) {
      const float2 st = row_stat[i];
      if (!(st.x > -INFINITY)) return 3;
      return __float_as_int(st.y) == x ? 0 : 1;
    }
    double px = ql::load_elem(a.target, target_at(i) + x, DT), qx = 1.0;
    if (stats) {
      if (!usable(row_stat[i]) || (has_q && !usable(row_stat[n + 1 + i]))) return 3;
      px = exp((px - row_stat[i].x) * a.inv_t) / zp;
    } else if (!(px < INFINITY)) {
      return 3;
    }
    if (has_q) {
      qx = ql::load_elem(a.draft, draft_at(i) + x, DT);
      if (stats) qx = exp((qx - row_stat[n + 1 + i].x) * a.inv_t) / zq;
      else if (!(qx < INFINITY)) return 3;
    }
    const double uq = u[i] * qx;
    if (stats && !exact && fabs(uq - px) <= 0x1p-14 * px) return 2;
    return uq < px ? 0 : 1;
  };
  int pos = 0, how = 0;
  for (;;) {
    if (warp == 0) {
      const int i = pos + lane;
      const int d = i < n ? decide(i, row_stat[min(i, kVerifyRows - 1)].y,
                                   row_stat[min(n + 1 + i, kVerifyRows - 1)].y, false)
                          : 1;
      const unsigned stop = __ballot_sync(0xffffffffu, d != 0);
      const int first = __ffs(stop) - 1;  // n - pos <= 31, so there is one
      const int what = __shfl_sync(0xffffffffu, d, first);
      if (lane == 0) {
        pos_s = pos + first;
        exact_s = what;
      }
    }
    __syncthreads();
    pos = pos_s;
    how = pos < n ? exact_s : 0;
    __syncthreads();
    if (how != 2) break;
    Row p{target_at(pos), row_stat[pos].x, 1.0};
    Row q{has_q ? draft_at(pos) : 0, has_q ? row_stat[n + 1 + pos].x : 0.f, 1.0};
    exact_sums(p, q, has_q);
    how = decide(pos, p.z, q.z, true);
    if (how != 0) break;
    ++pos;
  }
  // how: 0 all accepted (pos = n), 1 rejected at pos, 3 undecidable there
  const bool rejected = how == 1;
  bool bad = how == 3;
  if (stats && !bad) bad = greedy ? !(row_stat[pos].x > -INFINITY) : !usable(row_stat[pos]);
  if (rank == 0) {
    int32_t* tok = a.tokens + static_cast<size_t>(b) * (a.drafts + 1);
    for (int i = tid; i <= a.drafts; i += kVerifyThreads)
      if (i != pos || bad || greedy)
        tok[i] = i < pos ? ids[i]
                 : i == pos && greedy && !bad ? __float_as_int(row_stat[pos].y) : -1;
    if (tid == 0) a.accepted[b] = pos;
  }
  auto raise = [&]() {
    if (rank == 0 && tid == 0) {
      const bool id = pos < n && (ids[pos] < 0 || ids[pos] >= V);
      atomicOr(a.status, id ? ql::kStatusBadToken : ql::kStatusBadLogits);
    }
  };
  if (bad || greedy) {
    if (bad) raise();
    cluster_sync();  // nobody leaves while its shared memory may still be read
    return;
  }

  // ---- 3. the draw from the target's row, less the draft's after a rejection
  Row p{target_at(pos), stats ? row_stat[pos].x : 0.f, 1.0};
  const bool less_q = rejected && has_q;
  Row q{less_q ? draft_at(pos) : 0, less_q && stats ? row_stat[n + 1 + pos].x : 0.f, 1.0};
  exact_sums(p, q, less_q);
  const double rp = 1.0 / p.z, rq = 1.0 / q.z;
  const int out = rejected && !has_q ? ids[pos] : -1;  // a certain draft: its id is taken out
  bool less = rejected;
  auto left = [&](const int(&i)[4], double (&w)[4]) {  // whole warps
    weights(a.target, p, i, w);
    double v[4];
    if (less && less_q) weights(a.draft, q, i, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] *= rp;
      if (less) w[e] = less_q ? w[e] - v[e] * rq : i[e] == out ? 0.0 : w[e];
      w[e] = w[e] < 0 ? 0.0 : w[e];  // NaN stays
    }
  };
  // this lane's sum over its warp's part of [from, to)
  auto part_sum = [&](int from, int to) {
    double s = 0;
    each(from, to, [&](const int(&i)[4], int of) {
      double w[4];
      left(i, w);
#pragma unroll
      for (int e = 0; e < 4; ++e) s += e < of ? w[e] : 0.0;
    });
    return s;
  };
  double total = part_sum(lo, hi), unused = 0;
  double of_cta = cluster_sums(total, unused);
  if (less && total <= 0) {  // nothing left of the difference: the target itself
    less = false;
    total = part_sum(lo, hi);
    unused = 0;
    of_cta = cluster_sums(total, unused);
  }
  if (!(total > 0 && total < INFINITY)) {  // probabilities that are none
    raise();
    if (rank == 0 && tid == 0) a.tokens[static_cast<size_t>(b) * (a.drafts + 1) + pos] = -1;
    cluster_sync();
    return;
  }
  const double th = u[n] * total;
  // Of the lanes' shares (in lane order), the first where the running sum reaches
  // th, else the last that is not empty; `before` becomes the sum before it.
  auto find = [&](double v, double& before) {
    double cum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double w = __shfl_up_sync(0xffffffffu, cum, o);
      if (lane >= o) cum += w;
    }
    const unsigned some = __ballot_sync(0xffffffffu, v > 0);
    const unsigned hit = __ballot_sync(0xffffffffu, v > 0 && before + cum >= th);
    const int k = hit ? __ffs(hit) - 1 : some ? 31 - __clz(some) : 0;
    before += __shfl_sync(0xffffffffu, cum - v, k);
    return k;
  };
  double before = 0;
  const int owner = find(of_cta, before);
  cluster_sync();
  if (owner != rank) return;
  // sums[0] holds this CTA's warps' sums of the last part_sum
  int from = lo, to = hi;
  for (;;) {
    const int w = find(lane < kVerifyWarps ? sums[0][lane] : 0.0, before);
    const int f = warp_part(from, to, w), e = warp_part(from, to, w + 1);
    from = f;
    to = e;
    if (to - from <= 32) break;
    const double s = warp_total(part_sum(from, to));
    __syncthreads();
    if (lane == 0) sums[0][warp] = s;
    __syncthreads();
  }
  if (warp == 0) {
    const int at = min(min(from + lane, max(to - 1, from)), V - 1);
    const int i[4] = {at, at, at, at};
    double w[4];
    left(i, w);
    const double v = from + lane < to ? w[0] : 0.0;
    const unsigned some = __ballot_sync(0xffffffffu, v > 0);
    const int k = find(v, before);
    if (lane == 0)
      a.tokens[static_cast<size_t>(b) * (a.drafts + 1) + pos] = some ? from + k : -1;
  }
}

// CTAs of a cluster: up to 16 while the clusters together have an SM for each CTA, and
// a CTA has 1024 ids or more of its rows.
int cluster_ctas(int batch, int vocab, int num_sms) {
  int c = kMaxCluster;
  while (c > 1 && (static_cast<long long>(batch) * c > num_sms || vocab / c < 1024)) c /= 2;
  return c;
}

template <int DT>
cudaError_t launch_verify(const VerifyArgs& a, int batch, int num_sms, cudaStream_t s) {
  const int ctas = cluster_ctas(batch, a.vocab, num_sms);
  cudaError_t e = cudaSuccess;
  if (ctas > 8)
    e = cudaFuncSetAttribute(verify_kernel<DT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch) * ctas);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, verify_kernel<DT>, a);
}

}  // namespace

extern "C" int ql_verify_drafts(ql_ctx* c, const ql_verify_args* args) {
  if (!c || !args) return ql_fail(QL_ERR_INVALID, "ql_verify_drafts: NULL argument");
  const ql_verify_args& f = *args;
  if (f.batch < 0) return ql_fail(QL_ERR_INVALID, "batch %d is negative", f.batch);
  if (f.drafts < 0 || f.drafts > QL_VERIFY_MAX_DRAFTS)
    return ql_fail(QL_ERR_INVALID, "drafts %d must lie in [0, %d]", f.drafts, QL_VERIFY_MAX_DRAFTS);
  if (f.vocab <= 0) return ql_fail(QL_ERR_INVALID, "Verification requires a non-empty vocabulary");
  if (f.vocab > (1 << 22))
    return ql_fail(QL_ERR_UNSUPPORTED, "vocabulary of %d exceeds the device sampler's limit",
                   f.vocab);
  if (f.dtype != QL_F32 && f.dtype != QL_F16 && f.dtype != QL_BF16)
    return ql_fail(QL_ERR_INVALID, "unsupported element type %d", f.dtype);
  if (f.form != QL_VERIFY_LOGITS && f.form != QL_VERIFY_PROBS)
    return ql_fail(QL_ERR_INVALID, "unknown form %d", f.form);
  const bool probs = f.form == QL_VERIFY_PROBS;
  if (!probs && !std::isfinite(f.temperature))
    return ql_fail(QL_ERR_INVALID, "Sampler temperature must be finite, got %g",
                   static_cast<double>(f.temperature));
  const int64_t ts = f.target_stride ? f.target_stride : f.vocab;
  const int64_t ds = f.draft_stride ? f.draft_stride : f.vocab;
  if (ts < f.vocab || ds < f.vocab)
    return ql_fail(QL_ERR_INVALID, "a row stride is smaller than the vocabulary %d", f.vocab);
  if (f.batch == 0) return QL_OK;
  const bool greedy = !probs && f.temperature <= 0.f;
  if (!f.target || !f.tokens || !f.accepted || (f.drafts > 0 && !f.draft_ids) ||
      (!greedy && !f.uniforms))
    return ql_fail(QL_ERR_INVALID, "ql_verify_drafts: NULL buffer");
  const size_t eb = f.dtype == QL_F32 ? 4 : 2;
  auto off = [](const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; };
  if (off(f.target, eb) || off(f.draft, eb) || off(f.draft_ids, 4) || off(f.n_draft, 4) ||
      off(f.uniforms, 8) || off(f.tokens, 4) || off(f.accepted, 4))
    return ql_fail(QL_ERR_INVALID, "ql_verify_drafts: a buffer is not aligned to its element size");
  ql_device_guard dev(c->device);
  QLV_CUDA(dev.error(), "set device");
  VerifyArgs a{};
  a.target = f.target;
  a.draft = f.draft;
  a.ids = f.draft_ids;
  a.n_draft = f.n_draft;
  a.uniforms = f.uniforms;
  a.tokens = f.tokens;
  a.accepted = f.accepted;
  a.status = c->status;
  a.target_stride = ts;
  a.draft_stride = ds;
  a.drafts = f.drafts;
  a.vocab = f.vocab;
  a.dtype = f.dtype;
  a.probs = probs;
  a.inv_t = probs ? 1.0 : greedy ? 0.0 : 1.0 / static_cast<double>(f.temperature);
  cudaError_t e;
  if (f.dtype == QL_F32) e = launch_verify<ql::kF32>(a, f.batch, c->num_sms, c->stream);
  else if (f.dtype == QL_F16) e = launch_verify<ql::kF16>(a, f.batch, c->num_sms, c->stream);
  else e = launch_verify<ql::kBF16>(a, f.batch, c->num_sms, c->stream);
  QLV_CUDA(e, "launch the draft verification");
  return QL_OK;
}
