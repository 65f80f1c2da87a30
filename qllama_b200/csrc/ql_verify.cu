// ql_verify.cu -- verification of drafted tokens (qllama_model.h): speculative
// sampling's acceptance and the draw of the next token, beside ql_sample.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "../../include/qllama_model.h"
#include "ql_device.cuh"
#include "ql_internal.h"

namespace {

#define QLV_CUDA(call, what)                                                      \
  do {                                                                            \
    cudaError_t e_ = (call);                                                      \
    if (e_ != cudaSuccess) {                                                      \
      cudaGetLastError(); /* not the next launch's error */                       \
      return ql_fail(QL_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e_));        \
    }                                                                             \
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
  double exp_scale;  // 32 / (T ln2)
  double exp_least;  // -690 T: an exponential below exp(-690) is taken as 0
  float exp2_scale;  // 1 / (T ln2)
};

// One cluster of CTAs per sequence, each CTA with its share of every row.
//   1. f32 (maximum, sum of exponentials) of all of the sequence's rows at once --
//      the one pass over the logits, bound by their bytes.  (Greedy: largest logit and
//      its id.)
//   2. Every draft is decided from its two logits and those sums.  A decision whose
//      two sides are within 2^-14 of each other, far more than the f32 error, or below
//      f32's range is taken again from f64 sums of its rows, p and q being f64 numbers.
//   3. The draw compares running sums over the whole vocabulary with a threshold,
//      where an error of 1e-7 would change one token in some thousands: its sums are
//      f64, of the rows' weights wp, wq = exp((logit - maximum) / T).  After a rejected
//      draft the ids with wp / sum wp > wq / sum wq keep the difference.  Which they
//      are is decided with the f32 sums, so that one pass gives the whole sums and
//      those of the ids that count, and from them the sum of what is left: an id that
//      the f32 sums misjudge has a difference of 1e-6 of its probability or less, and
//      few have (when less than 1/32 is left, more may: a second pass then goes by the
//      f64 sums).  The threshold is looked for in the CTAs, the warps and the lanes in
//      turn.
// The CTAs of a cluster tell each other their sums by stores into one another's
// shared memory that count on an mbarrier there; all make the same decisions from the
// same numbers.  Nothing is kept outside shared memory.  A CTA whose wait for the others
// runs out writes -1 for the sequence and stays until they are at their end, so that no
// store of theirs meets shared memory that is no longer its own; the others have all
// that was sent to them when they leave.
// A small call is bound by the latencies of its steps, one after the other (32
// sequences, one row of 32000: 24 us with every warp following every decision, 17 us
// with the weights computed anew at every turn of the search).  So one loop takes all
// f64 sums, warp 0 alone decides what is next, and where a CTA's share is small
// enough its weights stay in shared memory for the search.  Greedy, logits and
// probabilities are kernels of their own, and rows are read in whole aligned groups
// with the odd ends on the side.
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
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float warp_max(float v) {  // NaN only of NaNs
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ double shfl_xor(double v, int o) {
  return __shfl_xor_sync(0xffffffffu, v, o);
}
// Sums of four values over the warp, each step halving what a lane still carries:
// lanes 8 i .. 8 i + 7 get the sum of v[i].
__device__ __forceinline__ double warp_totals(const double (&v)[4]) {
  const int lane = threadIdx.x & 31;
  const bool hi = lane & 16, up = lane & 8;
  const double a = (hi ? v[2] : v[0]) + shfl_xor(hi ? v[0] : v[2], 16);
  const double b = (hi ? v[3] : v[1]) + shfl_xor(hi ? v[1] : v[3], 16);
  double t = (up ? b : a) + shfl_xor(up ? a : b, 8);
  t += shfl_xor(t, 4);
  t += shfl_xor(t, 2);
  return t + shfl_xor(t, 1);
}
// A wait that looks often before it looks at the clock.  False, with the status raised,
// when the time ran out.
__device__ __forceinline__ bool await(uint64_t* bar, uint32_t parity, uint32_t* status) {
  for (int i = 0; i < 64; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(ql::smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return ql::mbar_wait_cluster(bar, parity, status);
}
__device__ __forceinline__ void st_async_f64(uint32_t remote_addr, double v, uint32_t remote_bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(
                   remote_addr),
               "l"(__double_as_longlong(v)), "r"(remote_bar)
               : "memory");
}

// exp((x - m) / T) in f64 for x <= m by the table method (P. T. P. Tang, 1989):
// (x - m) / T = (k + r) ln2 / 32 with |r| <= 1/2, k = 32 e + j; the result is
// 2^e 2^(j/32) exp(r ln2 / 32), the last by four terms of its series (the fifth is
// below 1.3e-12).  Lane j holds 2^(j/32), read by shuffles: whole warps call this.
struct Exp64 {
  double table, scale;
  // Differences x - m below it (an exponential under 1e-299) give 0.  They are compared
  // as they are, in f64: m + least in f32 may be a step of the logits too low, where
  // 2^e no longer is a number of the type.
  double least;
  __device__ __forceinline__ double operator()(float x, double m) const {
    return at(static_cast<double>(x) - m);
  }
  // the square of half the exponent's: down to f64's smallest numbers
  __device__ __forceinline__ double all(float x, double m) const {
    const double h = at(0.5 * (static_cast<double>(x) - m));
    return h * h;
  }
  __device__ __forceinline__ double at(double d) const {
    constexpr double L = 0.693147180559945309417232 / 32.0;
    constexpr double magic = 6755399441055744.0;  // 1.5 * 2^52
    const double t = fma(d, scale, magic);
    const int k = __double2loint(t);
    const double r = fma(d, scale, magic - t);
    double p = fma(r, L * L * L * L / 24, L * L * L / 6);
    p = fma(p, r, L * L / 2);
    p = fma(p, r, L);
    p = fma(p, r, 1.0);
    const int hi = __shfl_sync(0xffffffffu, __double2hiint(table), k) + ((k & ~31) << 15);
    const int lo = __shfl_sync(0xffffffffu, __double2loint(table), k);
    return d < least ? 0.0 : p * __hiloint2double(hi, lo);
  }
};

enum VerifyMode : int { kGreedy = 0, kLogits = 1, kProbs = 2 };

template <int DT>
__device__ __forceinline__ float half_word(uint32_t w, int upper) {
  if constexpr (DT == ql::kF16)
    return __half2float(__ushort_as_half(static_cast<uint16_t>(w >> (16 * upper))));
  return __uint_as_float(upper ? w & 0xffff0000u : w << 16);
}

// What the CTA does next: set by warp 0, read by all.
struct VerifyStep {
  int what;       // the sums to take, or kDone
  int from, to;   // over these ids
  int pos;        // of these rows
  int out;        // a certain draft's id that is taken out of the row, or -1
  double ratio;   // ids count where wp > ratio wq
  double fp, fq;  // and weigh wp fp - wq fq
};
// With sums: of the rows at a close decision, of what is left, of a part of it; without:
// that decision by its sums, the decisions from pos on, the end.
enum : int { kTotals = 0, kAtDraft, kLeft, kNarrow, kBegin, kGiveUp, kDone };

// T threads: 1024 where a cluster's CTAs have an SM each, 256 where three share one.
template <int DT, int MODE, int T>
__global__ void __launch_bounds__(T, T == 1024 ? 1 : 3) verify_kernel(const VerifyArgs a) {
  constexpr int kVerifyThreads = T, kVerifyWarps = T / 32;
  constexpr int kN = DT == ql::kF32 ? 4 : 8;  // elements of a 16-byte group
  constexpr int kLoads = 4;                   // groups of a lane in a piece
  constexpr uint32_t kNone = DT == ql::kF32 ? 0xff800000u : DT == ql::kF16 ? 0xfc00fc00u : 0xff80ff80u;
  __shared__ float2 part[kVerifyRows][kVerifyWarps];     // a row's (m, s) or (best, id) by warp
  __shared__ __align__(16) float2 from_cta[kVerifyRows][kMaxCluster];  // by CTA of the cluster
  __shared__ float2 row_stat[kVerifyRows];               // of the whole row
  __shared__ double sums[4][kVerifyWarps];
  __shared__ double sums_of[2][4][kMaxCluster];  // of each CTA, two turns
  constexpr int kKeep = T == 1024 ? 2048 : 4096;
  __shared__ double kept[MODE == kGreedy ? 1 : kKeep];  // weights of a share's ids
  __shared__ VerifyStep next_step;
  __shared__ __align__(8) uint64_t bars[3];
  __shared__ double pow2_32[32];                         // 2^(j/32)
  __shared__ int32_t id_of[QL_VERIFY_MAX_DRAFTS + 1];    // the drafts
  __shared__ double u_of[QL_VERIFY_MAX_DRAFTS + 1];
  __shared__ int lost;  // a wait for the other CTAs ran out
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = a.vocab;
  const int rank = static_cast<int>(cluster_rank()), ctas = static_cast<int>(cluster_size());
  const int b = blockIdx.x / ctas;
  if (tid == 0) {
    lost = 0;
    for (uint64_t& bar : bars) ql::mbar_init(&bar, 1);
    ql::fence_mbar_init();
  }
  if (MODE == kLogits && warp == 1) pow2_32[lane] = exp2(lane / 32.0);
  __syncthreads();
  ql::cluster_arrive_relaxed();
  ql::cluster_wait();  // every CTA's barriers are there
  ql::griddep_wait();
  ql::griddep_launch_dependents();
  const int n = a.n_draft ? min(max(a.n_draft[b], 0), a.drafts) : a.drafts;
  const int32_t* const ids = id_of;
  const double* const u = u_of;
  const bool has_q = MODE != kGreedy && a.draft != nullptr;
  // Row r: 0 .. n the target's, n + 1 .. 2n the draft's.
  constexpr size_t kBytes = DT == ql::kF32 ? 4 : 2;
  auto row_at = [&](int r) {
    return r <= n ? static_cast<const char*>(a.target) +
                        (static_cast<size_t>(b) * (a.drafts + 1) + r) * a.target_stride * kBytes
                  : static_cast<const char*>(a.draft) +
                        (static_cast<size_t>(b) * a.drafts + r - n - 1) * a.draft_stride * kBytes;
  };
  // Warp 0's lane i: the logits (probabilities) of draft i, ready when the rows' sums are.
  float drafted_p = 0.f, drafted_q = 0.f;
  if (warp == 0) {
    const int x = lane < n ? a.ids[static_cast<size_t>(b) * a.drafts + lane] : -1;
    if (lane < n) id_of[lane] = x;
    if (MODE != kGreedy && lane <= n)
      u_of[lane] = a.uniforms[static_cast<size_t>(b) * (a.drafts + 1) + lane];
    if (MODE != kGreedy && x >= 0 && x < V) {
      drafted_p = ql::load_elem(row_at(lane), x, DT);
      if (has_q) drafted_q = ql::load_elem(row_at(n + 1 + lane), x, DT);
    }
    __syncwarp();
  }
  // ---- 1.
  const float c = a.exp2_scale;
  if constexpr (MODE != kProbs) {
    const int nrows = n + 1 + (has_q ? n : 0);
    const float2 none = make_float2(-INFINITY, MODE == kGreedy ? __int_as_float(INT_MAX) : 0.f);
    for (int i = tid; i < nrows * kVerifyWarps; i += kVerifyThreads) part[0][i] = none;
    __syncthreads();
    // pieces of 32 * kLoads groups of this CTA's share of each row, by warps in turn
    const int span = (V / kN + ctas - 1) / ctas;
    const int pieces = max(1, (span + 32 * kLoads - 1) / (32 * kLoads));
    const int items = pieces * nrows;
    int it = static_cast<int>(static_cast<long long>(items) * warp / kVerifyWarps);
    const int end = static_cast<int>(static_cast<long long>(items) * (warp + 1) / kVerifyWarps);
    int row = it / pieces, piece = it % pieces;  // of the next piece to load
    uint4 now[kLoads], next[kLoads];
    int first = 0;  // id of the lane's first element of `next`
    float end_x = -INFINITY;  // an element outside the row's whole groups
    int end_id = 0;
    auto load = [&]() {
      const char* p = row_at(row);
      const int lead = static_cast<int>((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / kBytes);
      const int head = min(lead, V), groups = (V - head) / kN;
      const int g0 = rank * span + piece * 32 * kLoads + lane;
      const int stop = min(groups, (rank + 1) * span);
      const uint4* gp = reinterpret_cast<const uint4*>(p + head * kBytes);
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        next[j] = g0 + 32 * j < stop ? gp[g0 + 32 * j] : make_uint4(kNone, kNone, kNone, kNone);
      first = head + g0 * kN;
      end_x = -INFINITY;
      if (rank == 0 && piece == 0) {  // the ends: lanes 0-15 before, 16-31 behind
        end_id = lane < 16 ? lane : head + groups * kN + lane - 16;
        if (lane < 16 ? lane < head : end_id < V) end_x = ql::load_elem(p, end_id, DT);
      }
    };
    if (it < end) load();
    while (it < end) {
      const int at = row;
      float m = -INFINITY, s = 0.f;
      int best = INT_MAX, bad = 0;
      do {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) now[j] = next[j];
        const float ex = end_x;
        const int eid = end_id, id0 = first;
        if (++piece == pieces) {
          piece = 0;
          ++row;
        }
        if (++it < end) load();  // in flight while this piece is summed
        auto element = [&](int k) {
          const uint4 v = now[k / kN];
          const int e = k % kN, w = DT == ql::kF32 ? e : e / 2;
          const uint32_t x = w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w;
          if constexpr (DT == ql::kF32) return __uint_as_float(x);
          else return half_word<DT>(x, e & 1);
        };
        float top = ex;
#pragma unroll
        for (int k = 0; k < kLoads * kN; ++k) top = max_nan(top, element(k));
        if constexpr (MODE == kGreedy) {
          // a piece that matters is looked through again for its first largest
          bad |= !(top < INFINITY);
          if (top > m || (top == m && top > -INFINITY)) {
            int id = ex == top ? eid : INT_MAX;
#pragma unroll 1
            for (int j = kLoads - 1; j >= 0; --j) {
              const uint4 v = j == 0 ? now[0] : j == 1 ? now[1] : j == 2 ? now[2] : now[3];
              const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int e = kN - 1; e >= 0; --e) {
                float x;
                if constexpr (DT == ql::kF32) x = __uint_as_float(w[e]);
                else x = half_word<DT>(w[e / 2], e & 1);
                const int i = id0 + j * (32 * kN) + e;
                if (x == top && i < id) id = i;
              }
            }
            best = top > m ? id : min(best, id);
            m = top;
          }
        } else {
          top = fmaxf(top, m);  // a NaN is met again below
          // nothing above -inf yet: 0 for the maximum leaves zeros, and NaN a NaN
          const float ref = top > -INFINITY ? top : 0.f;
          s = s * exp2_fast(m == -INFINITY ? 0.f : (m - ref) * c) + exp2_fast((ex - ref) * c);
          m = top;
          float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < kLoads * kN; ++k) add[k % 4] += exp2_fast((element(k) - ref) * c);
          s += (add[0] + add[1]) + (add[2] + add[3]);
        }
      } while (it < end && row == at);
      // this warp's part of the row
      if constexpr (MODE == kGreedy) {
        const float top = warp_max(m);
        best = __reduce_min_sync(0xffffffffu, m == top ? best : INT_MAX);
        m = top;
        if (__any_sync(0xffffffffu, bad)) m = NAN;
        if (lane == 0) part[at][warp] = make_float2(m, __int_as_float(best));
      } else {
        const float top = warp_max(m);
        s *= m == top ? 1.f : m == -INFINITY ? 0.f * s : exp2_fast((m - top) * c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) part[at][warp] = make_float2(top, s);
      }
    }
    // (m, s) or (best, id) of the parts of a row that a warp's lanes hold: first of
    // the CTA's warps, told to every CTA, then of the CTAs
    if (tid == 0) ql::mbar_arrive_expect_tx(&bars[0], static_cast<uint32_t>(nrows * ctas * 8));
    __syncthreads();
#pragma unroll 1
    for (int turn = 0; turn < 2; ++turn) {
      if (turn == 1 && !__all_sync(0xffffffffu, await(&bars[0], 0, a.status))) {
        lost = 1;
        break;
      }
#pragma unroll 1
      for (int r = warp; r < nrows; r += kVerifyWarps) {
        float2 z = none;
        if (turn == 0 && lane < kVerifyWarps) z = part[r][lane];
        if (turn == 1 && lane < ctas) z = from_cta[r][lane];
        if constexpr (MODE == kGreedy) {  // a NaN marks the row
          const bool bad = __any_sync(0xffffffffu, z.x != z.x);
          const float top = warp_max(z.x);
          const int id = __reduce_min_sync(0xffffffffu, z.x == top ? __float_as_int(z.y) : INT_MAX);
          z = make_float2(bad ? NAN : top, __int_as_float(id));
        } else {  // sums under a maximum of -inf are zeros, or a NaN that marks the row
          const float top = warp_max(z.x);
          float s = z.x == top ? z.y : z.x == -INFINITY ? 0.f * z.y : z.y * exp2_fast((z.x - top) * c);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          z = make_float2(top, s);
        }
        if (turn == 0) {
          if (lane < ctas)
            ql::st_async_v2(ql::mapa_shared(ql::smem_u32(&from_cta[r][rank]), lane), z,
                            ql::mapa_shared(ql::smem_u32(&bars[0]), lane));
        } else if (lane == 0) {
          row_stat[r] = z;
        }
      }
    }
    __syncthreads();
  }
  int32_t* const tok = a.tokens + static_cast<size_t>(b) * (a.drafts + 1);

  // ---- 2. Warp 0: the first draft that is not accepted, from `pos` on.
  // verdict: 0 none (pos = n), 1 rejected, 2 too close for f32 sums, 3 cannot be decided
  int pos = 0, verdict = 0;
  // whether a row's numbers are those of a distribution
  auto usable = [&](int r) {
    if (MODE == kProbs) return true;
    const float2 st = row_stat[r];
    return MODE == kGreedy ? st.x > -INFINITY
                           : st.y > 0.f && st.y < INFINITY && st.x > -INFINITY;
  };
  auto decide = [&]() {
    const int i = lane;  // drafts before pos are accepted already
    int d = i < pos ? 0 : i < n ? 3 : 1;
    const int x = i >= pos && i < n ? ids[i] : -1;
    if (x >= 0 && x < V && usable(i) && (!has_q || usable(n + 1 + i))) {
      if constexpr (MODE == kGreedy) {
        d = __float_as_int(row_stat[i].y) == x ? 0 : 1;
      } else {
        const float lp = drafted_p, lq = drafted_q;
        double px = lp, qx = has_q ? lq : 1.0;
        if constexpr (MODE == kLogits) {
          px = exp2_fast((lp - row_stat[i].x) * c) / row_stat[i].y;
          if (has_q) qx = exp2_fast((lq - row_stat[n + 1 + i].x) * c) / row_stat[n + 1 + i].y;
        }
        const double uq = u[i] * qx;
        d = uq < px ? 0 : 1;
        if (MODE == kLogits &&  // close, or so small that f32 may have lost it
            (!(fabs(uq - px) > 0x1p-14 * px) || px < 1e-30 || qx < 1e-30))
          d = 2;
        if (MODE == kProbs && !(px < INFINITY && qx < INFINITY)) d = 3;
      }
    }
    pos = __ffs(__ballot_sync(0xffffffffu, d != 0)) - 1;  // n <= 31: lane n has one
    d = __shfl_sync(0xffffffffu, d, pos);
    verdict = pos < n ? d : 0;
    if (verdict != 3 && !usable(pos)) verdict = 3;
  };
  // Everything but the new token, which is `token` if that is known already.
  auto write = [&](bool known, int token) {
    if (rank != 0) return;
    for (int i = lane; i <= a.drafts; i += 32)
      if (i != pos || known) tok[i] = i < pos ? ids[i] : i == pos ? token : -1;
    if (lane == 0) a.accepted[b] = pos;
  };
  auto raise = [&]() {
    if (rank == 0 && lane == 0) {
      const bool id = pos < n && (ids[pos] < 0 || ids[pos] >= V);
      atomicOr(a.status, id ? ql::kStatusBadToken : ql::kStatusBadLogits);
    }
  };
  if constexpr (MODE == kGreedy) {
    if (warp == 0 && !lost) {
      decide();
      write(true, verdict == 3 ? -1 : __float_as_int(row_stat[pos].y));
      if (verdict == 3) raise();
    }
  } else if (MODE == kProbs || !lost) {
    // ---- 3.
    const int lo = static_cast<int>(static_cast<long long>(V) * rank / ctas);
    const int hi = static_cast<int>(static_cast<long long>(V) * (rank + 1) / ctas);
    const Exp64 ex{pow2_32[lane], a.exp_scale, a.exp_least};
    // warp 0's: sums of the rows at pos, the threshold, the sum before [from, to)
    double zp = 1.0, zq = 1.0, th = 0.0, before = 0.0;
    int turn = 0;
    if (tid == 0) next_step = {kBegin, lo, hi, 0, -1, 0.0, 1.0, 0.0};
#pragma unroll 1
    for (;;) {
      __syncthreads();
      VerifyStep z = next_step;
      if (z.what == kDone) break;
      auto share = [&](int w) {
        return z.from + static_cast<int>(static_cast<long long>(z.to - z.from) * w / kVerifyWarps);
      };
      const bool with_q = has_q && z.pos < n;
      const bool keep = z.to - z.from <= (with_q ? kKeep / 2 : kKeep);
      // of the ids that count: sums of wp, wq; of all
      if (z.what < kBegin) {
        double s[4] = {0.0, 0.0, 0.0, 0.0};
        const char* const prow = row_at(z.pos);
        const char* const qrow = row_at(with_q ? n + 1 + z.pos : z.pos);
        const float pm = MODE == kLogits ? row_stat[z.pos].x : 0.f;
        const float qm = MODE == kLogits && with_q ? row_stat[n + 1 + z.pos].x : 0.f;
        const int f = share(warp), e = share(warp + 1);
        constexpr int kIds = 4;  // of a lane at a time, their loads in flight together
        constexpr float kEmpty = MODE == kLogits ? -INFINITY : 0.f;
#pragma unroll 1
        for (int i0 = f + lane; i0 - lane < e; i0 += 32 * kIds) {
          float xp[kIds], xq[kIds];
#pragma unroll
          for (int k = 0; k < kIds; ++k) xp[k] = ql::load_elem(prow, min(i0 + 32 * k, e - 1), DT);
          if (with_q) {
#pragma unroll
            for (int k = 0; k < kIds; ++k) xq[k] = ql::load_elem(qrow, min(i0 + 32 * k, e - 1), DT);
          }
          double wp[kIds], wq[kIds];
#pragma unroll
          for (int k = 0; k < kIds; ++k) {
            const float x = i0 + 32 * k < e ? xp[k] : kEmpty;
            wp[k] = MODE == kLogits ? ex(x, pm) : static_cast<double>(x);
            wq[k] = 0.0;
          }
          if (with_q) {
#pragma unroll
            for (int k = 0; k < kIds; ++k) {
              const float x = i0 + 32 * k < e ? xq[k] : kEmpty;
              wq[k] = MODE == kLogits ? ex(x, qm) : static_cast<double>(x);
            }
          }
#pragma unroll
          for (int k = 0; k < kIds; ++k) {
            const bool counts = wp[k] > z.ratio * wq[k] && i0 + 32 * k != z.out;
            s[2] += wp[k];
            s[3] += wq[k];
            if (!counts) wp[k] = wq[k] = 0.0;
            s[0] += wp[k];
            s[1] += wq[k];
            if (keep && i0 + 32 * k < e) {
              kept[i0 + 32 * k - z.from] = wp[k];
              if (with_q) kept[kKeep / 2 + i0 + 32 * k - z.from] = wq[k];
            }
          }
        }
        const double t = warp_totals(s);
        if (lane % 8 == 0) sums[lane / 8][warp] = t;
      }
      __syncthreads();
      if (warp != 0) continue;

      // ---- warp 0: what these sums mean, and what is next
      bool draw = false, search = z.what == kNarrow;
      int what = kDone;
      if (z.what == kBegin) {
        decide();
        z.pos = pos;
        if (verdict == 2) what = kTotals;
        else if (verdict == 3) what = kGiveUp;
        else draw = true;
      } else if (z.what == kAtDraft) {  // (its own turn: 11.0 us for one sequence, 11.3 in the
        // branch that has the sums, where more values are held)
        double uq = u[pos];
        if (has_q)
          uq *= ex.all(__shfl_sync(0xffffffffu, drafted_q, pos), row_stat[n + 1 + pos].x) / zq;
        draw = !(uq < ex.all(__shfl_sync(0xffffffffu, drafted_p, pos), row_stat[pos].x) / zp);
        verdict = 1;
        if (!draw) {
          ++pos;
          what = kBegin;
        }
      } else if (z.what < kNarrow) {
        // lanes 8 i ..: sum i of the CTA
        double t = 0.0;
#pragma unroll
        for (int w = 0; w < kVerifyWarps; w += 8) t += sums[lane / 8][w + lane % 8];
        t += shfl_xor(t, 4);
        t += shfl_xor(t, 2);
        t += shfl_xor(t, 1);
        // the cluster's sums: a rank one exchange ahead writes the other turn's
        uint64_t* const bar = &bars[1 + (turn & 1)];
        if (lane == 0) ql::mbar_arrive_expect_tx(bar, static_cast<uint32_t>(32 * ctas));
        __syncwarp();
        const uint32_t mine = ql::smem_u32(&sums_of[turn & 1][lane / 8][rank]);
#pragma unroll
        for (int h = 0; h < kMaxCluster; h += 8)
          if (h + lane % 8 < ctas)
            st_async_f64(ql::mapa_shared(mine, h + lane % 8), t,
                         ql::mapa_shared(ql::smem_u32(bar), h + lane % 8));
        if (!__all_sync(0xffffffffu, await(bar, turn >> 1 & 1, a.status))) {
          if (lane == 0) {
            lost = 1;
            next_step.what = kDone;
          }
          continue;
        }
        t = 0.0;
#pragma unroll
        for (int h = 0; h < kMaxCluster; h += 8)
          if (h + lane % 8 < ctas) t += sums_of[turn & 1][lane / 8][h + lane % 8];
        t += shfl_xor(t, 4);
        t += shfl_xor(t, 2);
        t += shfl_xor(t, 1);  // lanes 8 i ..: sum i of the cluster
        const double inv = 1.0 / t;
        const double t2 = __shfl_sync(0xffffffffu, t, 16), t3 = __shfl_sync(0xffffffffu, t, 24);
        if (z.what == kTotals) {
          zp = t2;
          zq = t3;
          what = kAtDraft;
          z.to = z.from;
        } else {
          const bool less = z.fq != 0;
          if (less && MODE == kLogits) {
            z.fp = __shfl_sync(0xffffffffu, inv, 16);
            z.fq = __shfl_sync(0xffffffffu, inv, 24);
          }
          const double left = __shfl_sync(0xffffffffu, t, 0) * z.fp -
                              __shfl_sync(0xffffffffu, t, 8) * z.fq;
          th = u[n] * left;
          search = left > 0 && t2 < INFINITY && t3 < INFINITY;
          if (search && less && MODE == kLogits && left < 0.03125 && z.ratio != t2 / t3) {
            search = false;
            what = kLeft;
            z.ratio = t2 / t3;
            z.fp = z.fq = 1.0;
          } else if (!search) {
            what = kGiveUp;  // probabilities that are none, unless
            if ((less || z.out >= 0) && left <= 0) {  // the draft's took all: the target
              what = kLeft;
              z.out = -1;
              z.ratio = z.fq = 0.0;
              z.fp = 1.0;
            }
          }
        }
      }
      // Of the lanes' parts (in lane order), the first where the running sum reaches th,
      // else the last that is not empty; `before` becomes the sum before it.
      unsigned some = 0;
      auto find = [&](double part) {
        double cum = part;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, cum, o);
          if (lane >= o) cum += v;
        }
        some = __ballot_sync(0xffffffffu, part > 0);
        const unsigned hit = __ballot_sync(0xffffffffu, part > 0 && before + cum >= th);
        const int k = hit ? __ffs(hit) - 1 : some ? 31 - __clz(some) : 0;
        before += __shfl_sync(0xffffffffu, cum - part, k);
        return k;
      };
      if (search) {
        auto weigh = [&](double wp, double wq) { return wp * z.fp - wq * z.fq; };
        bool here = true;
        if (z.what == kLeft) {  // the CTA
          write(false, 0);
          const int at = (turn & 1) * 4 * kMaxCluster + lane;
          const double* const of = &sums_of[0][0][0];
          here = find(lane < ctas ? weigh(of[at], of[at + kMaxCluster]) : 0.0) == rank;
        }
        if (here) {  // its warp
          const int w = find(lane < kVerifyWarps ? weigh(sums[0][lane], sums[1][lane]) : 0.0);
          const int f = share(w), e = share(w + 1);
          if (keep) {  // the lane's ids of that warp, then the id
            auto kept_at = [&](int i) {
              return weigh(kept[i - z.from], with_q ? kept[kKeep / 2 + i - z.from] : 0.0);
            };
            const int len = ((e - f + 31) / 32) | 1;  // odd: no two lanes on one bank
            double v = 0.0;
            for (int j = 0; j < len; ++j) {
              const int i = f + lane * len + j;
              if (i < e) v += kept_at(i);
            }
            const int i0 = f + find(v) * len;
            const int k = find(lane < len && i0 + lane < e ? kept_at(i0 + lane) : 0.0);
            if (lane == 0) tok[pos] = some ? i0 + k : -1;
          } else {
            what = kNarrow;
            z.from = f;
            z.to = e;
          }
        }
      }
      turn += z.what == kTotals || z.what == kLeft;
      // What a rejected draft leaves of the target's row, or all of it.
      if (draw) {
        const bool less = verdict == 1 && has_q;
        what = kLeft;
        z.from = lo;
        z.to = hi;
        z.out = verdict == 1 && !has_q ? ids[pos] : -1;
        z.ratio = !less ? 0.0
                  : MODE == kProbs
                      ? 1.0
                      : static_cast<double>(row_stat[pos].y) / row_stat[n + 1 + pos].y;
        z.fp = 1.0;
        z.fq = less ? 1.0 : 0.0;
      }
      if (what == kGiveUp) {
        write(true, -1);
        raise();
        what = kDone;
      }
      z.what = what;
      z.pos = pos;
      if (what == kTotals || what == kBegin) {
        z.from = lo;
        z.to = hi;
      }
      if (what == kTotals) {
        z.out = -1;
        z.ratio = 0.0;
      }
      if (lane == 0) next_step = z;
    }
  }
  if (lost && warp == 0) {
    for (int i = lane; i <= a.drafts; i += 32) tok[i] = -1;
    if (lane == 0) a.accepted[b] = 0;
  }
  ql::cluster_arrive_relaxed();
  if (lost) ql::cluster_wait();
}

// CTAs of a cluster: up to 16, in powers of two, while all sequences' CTAs are not many
// more than run at once (three to an SM); 1024 ids or more each, or 4096 when the SMs
// are shared and the CTAs slow one another down (32 sequences, one row of 32000: 12.4 us
// with 8, 15.8 us with 16; 8 sequences of 6 rows: 15.9 us and 13.0 us).
int cluster_ctas(int batch, int vocab, int num_sms) {
  int c = kMaxCluster;
  while (c > 1) {
    const long long all = static_cast<long long>(batch) * c;
    if (all <= 4LL * num_sms && vocab / c >= (all > 2LL * num_sms ? 4096 : 1024)) break;
    c /= 2;
  }
  return c;
}

template <int DT, int MODE, int T>
cudaError_t launch_verify_as(const VerifyArgs& a, int batch, int ctas, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = ql_once_per_device(done, [] {
    return cudaFuncSetAttribute(verify_kernel<DT, MODE, T>,
                                cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch) * ctas);
  cfg.blockDim = dim3(T);
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
  return cudaLaunchKernelEx(&cfg, verify_kernel<DT, MODE, T>, a);
}

template <int DT, int MODE>
cudaError_t launch_verify_mode(const VerifyArgs& a, int batch, int num_sms, cudaStream_t s) {
  const int ctas = cluster_ctas(batch, a.vocab, num_sms);
  // a few clusters with long shares: four times the warps (two sequences of 8 rows of
  // 128000 f32 23.7 us, 26.1 us with 256 threads; one of 5 rows of 32000 16.0 us, 10.9 us)
  return batch * ctas <= num_sms / 2 && a.vocab / ctas >= 4096
             ? launch_verify_as<DT, MODE, 1024>(a, batch, ctas, s)
             : launch_verify_as<DT, MODE, 256>(a, batch, ctas, s);
}

template <int DT>
cudaError_t launch_verify(const VerifyArgs& a, int batch, int num_sms, cudaStream_t s) {
  if (a.probs) return launch_verify_mode<DT, kProbs>(a, batch, num_sms, s);
  return a.inv_t == 0 ? launch_verify_mode<DT, kGreedy>(a, batch, num_sms, s)
                      : launch_verify_mode<DT, kLogits>(a, batch, num_sms, s);
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
  // (1 / (T ln2) of a smaller one is no f32 number)
  if (!probs && f.temperature > 0.f && f.temperature < FLT_MIN)
    return ql_fail(QL_ERR_UNSUPPORTED, "temperature %g is positive, but below f32's normal range",
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
  a.exp_scale = a.inv_t * (32.0 / 0.693147180559945309417232);
  a.exp_least = -690.0 / a.inv_t;
  a.exp2_scale = static_cast<float>(a.inv_t / 0.693147180559945309417232);
  cudaError_t e;
  if (f.dtype == QL_F32) e = launch_verify<ql::kF32>(a, f.batch, c->num_sms, c->stream);
  else if (f.dtype == QL_F16) e = launch_verify<ql::kF16>(a, f.batch, c->num_sms, c->stream);
  else e = launch_verify<ql::kBF16>(a, f.batch, c->num_sms, c->stream);
  QLV_CUDA(e, "launch the draft verification");
  return QL_OK;
}
