// ql_verify.cu -- verification of drafted tokens (qllama_model.h): speculative
// sampling's acceptance and the draw of the next token, beside ql_sample.
#include <cuda_runtime.h>

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

constexpr int kVerifyThreads = 512;

__device__ double vsum(double v, double* red) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) t += red[i];
  return t;
}

__device__ float vmax(float v, float* red) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = red[0];
  for (int i = 1; i < static_cast<int>(blockDim.x >> 5); ++i) t = fmaxf(t, red[i]);
  return t;
}

// One row as a distribution: value(i) is its unnormalised weight, z the sum.
struct Row {
  const void* base;
  size_t at;
  int dtype;
  bool probs;
  float m;
  double inv_t, z;
  __device__ float raw(int i) const { return ql::load_elem(base, at + i, dtype); }
  __device__ double value(int i) const {
    const float x = raw(i);
    return probs ? x : exp((static_cast<double>(x) - m) * inv_t);
  }
};

// One CTA per sequence.
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const VerifyArgs a) {
  __shared__ double red[kVerifyThreads / 32];
  __shared__ double part[kVerifyThreads];
  __shared__ float redf[kVerifyThreads / 32];
  __shared__ int found_s;
  const int b = blockIdx.x, V = a.vocab, tid = threadIdx.x;
  const int n = a.n_draft ? min(max(a.n_draft[b], 0), a.drafts) : a.drafts;
  int32_t* tok = a.tokens + static_cast<size_t>(b) * (a.drafts + 1);
  const int32_t* ids = a.ids + static_cast<size_t>(b) * a.drafts;
  const double* u = a.uniforms ? a.uniforms + static_cast<size_t>(b) * (a.drafts + 1) : nullptr;
  for (int i = tid; i <= a.drafts; i += kVerifyThreads) tok[i] = -1;
  __syncthreads();
  auto open = [&](const void* base, size_t row, int64_t stride, bool& bad) {
    Row r{base, row * static_cast<size_t>(stride), a.dtype, a.probs != 0, 0.f, a.inv_t, 1.0};
    float m = -INFINITY;
    int wrong = 0;
    for (int i = tid; i < V; i += kVerifyThreads) {
      const float x = r.raw(i);
      wrong |= !(x < INFINITY);
      m = fmaxf(m, x);
    }
    wrong = __syncthreads_or(wrong);
    r.m = vmax(m, redf);
    bad = wrong || (a.probs ? !(r.m > 0.f) : r.m == -INFINITY);
    if (!a.probs && !bad && a.inv_t > 0) {
      double s = 0;
      for (int i = tid; i < V; i += kVerifyThreads) s += r.value(i);
      r.z = vsum(s, red);
    }
    return r;
  };
  int pos = 0;
  bool bad = false, rejected = false;
  Row p{}, q{};
  for (;; ++pos) {
    p = open(a.target, static_cast<size_t>(b) * (a.drafts + 1) + pos, a.target_stride, bad);
    if (bad || pos == n) break;
    const int x = ids[pos];
    bad = x < 0 || x >= V;
    if (bad) break;
    if (a.inv_t == 0) {
      if (tid == 0) found_s = V;
      __syncthreads();
      for (int i = tid; i < V; i += kVerifyThreads)
        if (p.raw(i) == p.m) {
          atomicMin(&found_s, i);
          break;
        }
      __syncthreads();
      rejected = found_s != x;
      __syncthreads();
      if (rejected) break;
    } else {
      double qx = 1.0;
      if (a.draft) {
        q = open(a.draft, static_cast<size_t>(b) * a.drafts + pos, a.draft_stride, bad);
        if (bad) break;
        qx = q.value(x) / q.z;
      }
      rejected = !(u[pos] * qx < p.value(x) / p.z);
      if (rejected) break;
    }
    if (tid == 0) tok[pos] = x;
  }
  if (tid == 0) a.accepted[b] = pos;
  if (bad) {
    if (tid == 0) {
      const bool id = pos < n && (ids[pos] < 0 || ids[pos] >= V);
      atomicOr(a.status, id ? ql::kStatusBadToken : ql::kStatusBadLogits);
    }
    return;
  }
  if (a.inv_t == 0) {
    if (tid == 0) found_s = V;
    __syncthreads();
    for (int i = tid; i < V; i += kVerifyThreads)
      if (p.raw(i) == p.m) {
        atomicMin(&found_s, i);
        break;
      }
    __syncthreads();
    if (tid == 0) tok[pos] = found_s;
    return;
  }
  const int x = rejected ? ids[pos] : -1;
  auto weight = [&](int i, bool less) {
    double w = p.value(i) / p.z;
    if (less) w = a.draft ? w - q.value(i) / q.z : (i == x ? 0.0 : w);
    return w > 0 ? w : 0.0;
  };
  // thread t sums the contiguous ids [t * per, (t + 1) * per)
  const int per = (V + kVerifyThreads - 1) / kVerifyThreads;
  for (int pass = 0; pass < 2; ++pass) {
    const bool less = rejected && pass == 0;
    double s = 0;
    for (int i = tid * per; i < min(V, (tid + 1) * per); ++i) s += weight(i, less);
    __syncthreads();
    part[tid] = s;
    __syncthreads();
    double total = 0;
    for (int t = 0; t < kVerifyThreads; ++t) total += part[t];
    if (!(total > 0) && less) continue;  // nothing left of the difference: the target itself
    if (tid == 0) {
      const double th = u[n] * total;
      double cum = 0;
      int last = -1, hit = -1;
      for (int t = 0; t < kVerifyThreads && hit < 0; ++t) {
        if (cum + part[t] < th && t + 1 < kVerifyThreads) {
          cum += part[t];
          continue;
        }
        for (int i = t * per; i < min(V, (t + 1) * per); ++i) {
          const double w = weight(i, less);
          if (w <= 0) continue;
          last = i;
          cum += w;
          if (cum >= th) {
            hit = i;
            break;
          }
        }
      }
      if (hit < 0)
        for (int i = V - 1; i >= 0 && last < 0; --i)
          if (weight(i, less) > 0) last = i;
      tok[pos] = hit >= 0 ? hit : last;
    }
    return;
  }
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
  verify_kernel<<<f.batch, kVerifyThreads, 0, c->stream>>>(a);
  QLV_CUDA(cudaGetLastError(), "launch the draft verification");
  return QL_OK;
}
