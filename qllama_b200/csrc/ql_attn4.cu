// ql_attn4.cu -- attention of a few query tokens over a Q4_0 cache for B200 (sm_100a).
//
// One KV head's 64 positions are one record of 72 hd bytes (Q4Record: codes of K and V, then
// their scales), so a tile comes into shared memory as one bulk copy.  The work is the list of
// all tiles of all jobs, a job being one (sequence, KV head, up to eight query rows: heads of
// the group, of several tokens where they fit).  Every CTA takes an equal run of that list and
// every warp of it an equal part, streaming its tiles through a ring of its own: no barrier
// between warps until the run is done, whatever the sequences' lengths.  A job that lies inside
// a warp's part is finished there; pieces of others are joined in the CTA, and across CTAs by
// the last one to arrive.
//
// Per 16 positions, on the tensor cores (m16n8k16, positions and value columns as rows, query
// rows as columns, so that no row of a fragment is idle):
//   S = K q^T      A = the K codes, B = q
//   O = V^T P      A = the V codes, B = P times the block's scale
// A code c masked out of its word is the f16 number c 2^-24 (or, in the next nibble, c 2^-20):
// f16's subnormals hold the codes exactly and the matrix instruction takes them as they are, so
// that a fragment register costs one AND.  The powers of two are folded into q and the output.
// A K scale multiplies the block's partial sums in f32, a V scale the probabilities in f16 (V's
// scales as they are, or times a power of two that keeps small ones' products out of f16's
// subnormals and large ones' below its overflow).  The
// 8 that is subtracted from every code enters S as the product of K's scales with -8 sum q of each
// block, and leaves O with the product of ones and the same rounded P d that the codes met, so
// that a rounding counts with the value and not with the code; ones and P give the sum of P.
//
// Bound by HBM for long caches (2304 bytes of a head_dim 128 cache per 16 positions against
// about 200 instructions of one warp): 8 sequences of 32768 positions, 32/8 heads, 302 MB, take
// 69 us, of which the stream of tiles is some 53 (5.7 TB/s) and the rest the beginning (look-ups
// and queries, about 3 us), the joining (3 to 5 us) and the launch.  From L2, as with drafted
// tokens whose jobs share the keys, it is bound by instruction issue: half of the ALU's slots.
// Other shapes of the kernel measured the same or slower: sixteen warps of 128 registers, one
// step of 16 positions, sixteen query rows a job.
#include <math_constants.h>

#include <algorithm>
#include <atomic>

#include "ql_append.cuh"
#include "ql_device.cuh"
#include "ql_internal.h"
#include "ql_kernels.cuh"

namespace ql {

namespace {

constexpr float kLog2e4 = 1.4426950408889634f;
// A probability is 2^arg with arg at most kTop: times a scale below 2 it is below f16's overflow.
// The reference it is relative to moves only when an arg exceeds that, by enough to leave kSlack
// free.  What is free is lost at the other end, where f16's subnormals begin 25 powers of two
// below: outputs of positions that are e^18 times less likely than another one without a value
// are 0.0005 of their norm off (with six bits free 0.003, and 8 x 32768 1 % faster; with one
// 0.0004 and 1 % slower).
constexpr float kTop = 14.f, kSlack = 3.f;
constexpr float kFused = 1 << 20;

template <int HD>
struct Attn4Cfg {
  static constexpr int kNb = HD / 32;
  static constexpr int kWarps = 12;
  static constexpr int kRecord = 72 * HD;
  static constexpr int kStages = HD == 128 ? 2 : 4;  // of a warp's ring, at most
  static constexpr int kPart = 8 * HD + 16;  // floats of a piece: rows, then (reference, sum)
  static constexpr size_t smem(int stages) {
    return 128 + static_cast<size_t>(kWarps) * stages * (kRecord + 8) + kWarps * 32 + 16;
  }
  static_assert(kPart * 4 <= kRecord, "a warp's last piece takes its ring's place");
};

// D = A B
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// m16n8k8: D = A B.
__device__ __forceinline__ void mma_f16_k8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, "
      "{%7,%7,%7,%7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b), "f"(0.f));
}

// The transpose of an 8 x 8 matrix of f16 held as pairs along its rows.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  const __half2 d = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}

__device__ __forceinline__ float ex2(float x) {  // 2^x; -inf -> +0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Orders this thread's stores to shared memory before later bulk copies into it.
__device__ __forceinline__ void fence_proxy_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// A probability's exponent, not fused: the reference was taken from a rounded product, and where
// that is above kFused, what the rounding left off would show.
__device__ __forceinline__ float exponent(float y, float f, float ref) {
  return __fsub_rn(__fmul_rn(y, f), ref);
}

__device__ __forceinline__ float half_of(const uint32_t& w, bool high) {
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return high ? __high2float(h) : __low2float(h);
}

// A job of the list: its sequence, KV head and query rows, and its tiles.
struct Job {
  int b, id, kvh, row0, rows;
  int t0, tiles;  // its first place in the list of tiles, and their number there
};

// a / b for 0 <= a < 2^30 and a quotient below 2^22, where the product with the reciprocal is at
// most one off (an integer division takes several times as long, and these stand one behind
// the other before the first key arrives).
__device__ __forceinline__ int divide(int a, int b) {
  int q = static_cast<int>(static_cast<float>(a) * __frcp_rn(static_cast<float>(b)));
  const int r = a - q * b;
  if (r < 0) --q;
  if (r >= b) ++q;
  return q;
}

// Places that a job of sequence b takes in the list: its tiles, or (aligned) as many as its CTAs
// take, the last ones empty.
__device__ __forceinline__ int seq_tiles(const Attn4Args& a, int b) {
  const int end = a.seqs.start[b] + a.new_len;
  const int n = a.sel ? sel_blocks(end - 1, a.sel_max) : (end + kTile - 1) / kTile;
  return a.aligned ? divide(n + a.per_cta - 1, a.per_cta) * a.per_cta : n;
}

// Job k of sequence b.
__device__ __forceinline__ Job job_of(const Attn4Args& a, int b, int k, int tiles) {
  Job j;
  j.b = b;
  j.tiles = tiles;
  j.t0 = a.first[b] + k * tiles;
  j.id = b * a.cache.hkv * a.units + k;
  j.kvh = divide(k, a.units);
  const int unit = k - j.kvh * a.units;
  if (a.sel) {  // a list belongs to one token: chunks of its heads
    const int per = (a.group + 7) / 8, t = divide(unit, per), h0 = (unit - t * per) * 8;
    j.row0 = t * a.group + h0;
    j.rows = min(8, a.group - h0);
  } else {
    j.row0 = unit * 8;
    j.rows = min(8, a.new_len * a.group - j.row0);
  }
  return j;
}

__device__ __forceinline__ Job job_at(const Attn4Args& a, int x) {
  int lo = 0, hi = a.batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.first[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  const int tiles = seq_tiles(a, lo);
  return job_of(a, lo, divide(x - a.first[lo], tiles), tiles);
}

// The job behind j (which is not the last one).
__device__ __forceinline__ Job next_job(const Attn4Args& a, const Job& j) {
  const int per = a.cache.hkv * a.units, k = j.id - j.b * per + 1;
  return k < per ? job_of(a, j.b, k, j.tiles) : job_of(a, j.b + 1, 0, seq_tiles(a, j.b + 1));
}

// The record that holds tile x of the list, of job j; -1 for a place behind the job's tiles (or
// behind a selection's blocks).
__device__ __forceinline__ int record_at(const Attn4Args& a, const Job& j, int x) {
  const CacheView& c = a.cache;
  int tile = x - j.t0;
  if (a.sel) {
    const int t = divide(j.row0, a.group);
    if (tile >= sel_blocks(a.seqs.start[j.b] + t, a.sel_max)) return -1;
    tile = a.sel[(static_cast<size_t>(j.b * a.new_len + t) * c.hkv + j.kvh) * a.sel_max + tile];
  } else if (tile * kTile >= a.seqs.start[j.b] + a.new_len) {
    return -1;
  }
  const int per = c.page / kTile;
  const int in_seq = per == 1 ? tile : tile / per;
  int page = c.block_table[static_cast<size_t>(a.seqs.seq[j.b]) * c.pages_per_seq + in_seq];
  if (page < 0 || page >= c.num_pages) {
    atomicOr(a.status, kStatusBadPage);
    page = 0;  // keep the pipeline consistent; the result is flagged
  }
  return (page * c.hkv + j.kvh) * per + tile - in_seq * per;
}

// Element offset of query row `row` (token row / group, head row % group) in q and out.
__device__ __forceinline__ size_t row_offset(const Attn4Args& a, const Job& j, int row, int hd) {
  const int t = divide(row, a.group), h = row - t * a.group;
  return ((static_cast<size_t>(j.b) * a.new_len + t) * a.hq + j.kvh * a.group + h) * hd;
}

}  // namespace

// LO: q enters as two f16 parts; not needed where it is of 16 bits and arrives rotated: scaled by
// its power of two it is left in steps of at most 2^-38 of the row's largest (of 2^-34 in the odd
// places, which enter divided by 16), and those of bf16's eight bits that lie above them, or of
// f16's eleven, are all there.
template <int HD, bool LO>
__global__ void __launch_bounds__(32 * Attn4Cfg<HD>::kWarps, 1)
    attn4_kernel(const __grid_constant__ Attn4Args a) {
  using C = Attn4Cfg<HD>;
  constexpr int NB = C::kNb, W = C::kWarps;
  const int S = a.stages, ring_bytes = S * C::kRecord;
  constexpr Q4Record kRec{HD};
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~static_cast<uintptr_t>(127));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  uint8_t* ring = smem + warp * ring_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + W * ring_bytes) + warp * S;
  // the last job of every warp's part, for the joining
  Job* last_job = reinterpret_cast<Job*>(smem + W * ring_bytes + W * S * 8);
  int* flag = reinterpret_cast<int*>(last_job + W);
  int* died = flag + 2;  // of a warp whose copy did not come in time: that tile
  static_assert(W * sizeof(Job) + (2 + W) * sizeof(int) <= W * 32 + 16, "smem()'s last part");

  const int c0 = blockIdx.x * a.per_cta, c1 = min(c0 + a.per_cta, a.total);
  const int w0 = min(c0 + warp * a.per_warp, c1), w1 = min(w0 + a.per_warp, c1);
  if (lane == 0) {
    for (int s = 0; s < S; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  // Before the previous kernel is waited for: the jobs of the first 32 tiles, and what is read
  // first is fetched into L2 (prefetches read nothing into the CTA; lines written meanwhile
  // are updated in L2).
  Job lane_job = job_at(a, min(w0 + lane, a.total - 1));
  Job job;  // of the part's first tile
  job.b = __shfl_sync(0xffffffffu, lane_job.b, 0);
  job.id = __shfl_sync(0xffffffffu, lane_job.id, 0);
  job.kvh = __shfl_sync(0xffffffffu, lane_job.kvh, 0);
  job.row0 = __shfl_sync(0xffffffffu, lane_job.row0, 0);
  job.rows = __shfl_sync(0xffffffffu, lane_job.rows, 0);
  job.t0 = __shfl_sync(0xffffffffu, lane_job.t0, 0);
  job.tiles = __shfl_sync(0xffffffffu, lane_job.tiles, 0);
  if (w0 < w1) {
    const int entry = (w0 + lane - lane_job.t0) / (a.cache.page / kTile);
    if (!a.sel && w0 + lane < w1 && entry < a.cache.pages_per_seq)  // (aligned: places without one)
      prefetch_l2(a.cache.block_table +
                  static_cast<size_t>(a.seqs.seq[lane_job.b]) * a.cache.pages_per_seq + entry);
    const int esize = a.in_dtype == kF32 ? 4 : 2;
    if (lane < job.rows * HD * esize / 128)
      prefetch_l2(static_cast<const char*>(a.q) +
                  (row_offset(a, job, job.row0 + lane * 128 / (HD * esize), HD) * esize +
                   lane * 128 % (HD * esize)));
  }
  griddep_wait();
  griddep_launch_dependents();

  // -------------------------------------------------------------- the ring --
  // The lanes hold the records of 32 tiles at a time; lane 0 issues.
  int lane_rec = w0 < w1 ? record_at(a, lane_job, min(w0 + lane, a.total - 1)) : -1;
  auto issue = [&](int i, int stage) {
    if ((i & 31) == 0 && i > 0) {
      const int x = min(w0 + i + lane, w1 - 1);
      lane_rec = record_at(a, job_at(a, x), x);
    }
    const int rec = __shfl_sync(0xffffffffu, lane_rec, i & 31);
    if (lane != 0) return;
    uint64_t* bar = &full[stage];
    if (rec < 0) {
      mbar_arrive(bar);
    } else {
      mbar_arrive_expect_tx(bar, C::kRecord);
      bulk_load(ring + stage * C::kRecord,
                static_cast<const uint8_t*>(a.cache.k) + static_cast<size_t>(rec) * kRec.bytes(),
                C::kRecord, bar);
    }
  };
  for (int i = 0; i < S && w0 + i < w1; ++i) issue(i, i);

  // This lane's places in a record: K codes and scales of position g, V's of the pair 2 tq.
  const int k_at = q4_k_byte(g, 8 * tq, NB);
  const int v_at = static_cast<int>(kRec.v_codes()) + q4_v_byte(2 * tq, 4 * g, NB);
  const int ks_at = static_cast<int>(kRec.k_scales()) + 2 * q4_k_scale(g, 0, NB);
  const int vs_at = static_cast<int>(kRec.v_scales()) + 2 * q4_v_scale(2 * tq, 0, NB);
  const int kw_at = ks_at + (NB == 4 ? (tq & 1) * 4 : 0);  // the scales of blocks 2 tq, 2 tq + 1
  constexpr uint32_t kOnes = 0x3c003c00u;  // two f16

  bool alive = true;
  int stage = 0, phase = 0;  // of the next tile
  int x = w0;
  while (x < w1) {
    if (x > w0) job = next_job(a, job);
    const int seg1 = min(w1, job.t0 + job.tiles);
    const int start = a.seqs.start[job.b];

    // ------------------------------------------------------------- q --
    // Lane (g, tq) holds dims 32 b + 8 tq .. + 7 of row g: the columns of B in the order in
    // which the K words' nibbles come out (j and j + 4 together; odd ones, whose codes are
    // 16 times as large, divided by 16).  Each row is scaled by a power of two to [2^14, 2^15):
    // far from f16's subnormals, and a 32nd of a block's sum stays in f16's range.
    uint32_t qh[NB][2][2], ql[NB][2][2], qo;
    float f[2];
    {
      float v[NB][8];
      const bool live = g < job.rows;
      const int row = job.row0 + (live ? g : 0);
      const size_t off = row_offset(a, job, row, HD) + 8 * tq;
      // the type is settled outside the loads, so that all are under way at once
      if (a.in_dtype == kF32 && a.q_vec) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + off);
        float4 w[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) w[b][0] = p[8 * b], w[b][1] = p[8 * b + 1];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          v[b][0] = w[b][0].x, v[b][1] = w[b][0].y, v[b][2] = w[b][0].z, v[b][3] = w[b][0].w;
          v[b][4] = w[b][1].x, v[b][5] = w[b][1].y, v[b][6] = w[b][1].z, v[b][7] = w[b][1].w;
        }
      } else if (a.in_dtype != kF32 && a.q_vec) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + off);
        uint4 w[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) w[b] = p[4 * b];
        const bool half = a.in_dtype == kF16;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t in[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&in[k]));
            v[b][2 * k] = half ? y.x : __uint_as_float(in[k] << 16);
            v[b][2 * k + 1] = half ? y.y : __uint_as_float(in[k] & 0xffff0000u);
          }
        }
      } else {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int k = 0; k < 8; ++k) v[b][k] = load_elem(a.q, off + 32 * b + k, a.in_dtype);
      }
      const double2* rope =
          a.rope_stride ? a.rope + static_cast<size_t>(start + divide(row, a.group)) * a.rope_stride
                        : nullptr;
      float mx = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int d = 32 * b + 8 * tq;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (!live) v[b][k] = 0.f;
        if (rope) {
#pragma unroll
          for (int k = 0; k < 8; k += 2)
            rope_pair(v[b][k], v[b][k + 1], rope[(d + k) / 2], v[b][k], v[b][k + 1]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) mx = fmaxf(mx, fabsf(v[b][k]));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const uint32_t bits = __float_as_uint(mx);
      int e = static_cast<int>(bits >> 23) - 127 - 14;
      if (bits == 0 || bits >= 0x7f800000u) e = 0;
      e = max(e, -100);
      const float down = pow2f(-e);
      float sums[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float s = 0.f;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float u = r ? down * 0.0625f : down;
            const float y0 = v[b][2 * ks + r] * u, y1 = v[b][2 * ks + r + 4] * u;
            float h0, l0, h1, l1;
            split16<false>(y0, h0, l0);
            split16<false>(y1, h1, l1);
            qh[b][ks][r] = pack2<false>(h0, h1);
            ql[b][ks][r] = pack2<false>(l0, l1);
            s += (LO ? y0 + y1 : h0 + h1) * (r ? 16.f : 1.f);
          }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        sums[b] = s * -0.03125f;  // -8 times it, by 2^8
      }
      // B of the K scales' product: column g, the sums' high parts under blocks 2 tq, 2 tq + 1
      // and what is left of them under the same scales again
      const bool low = NB == 4 ? tq >= 2 : tq == 1;
      float pair[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float s = NB == 4 && (tq & 1) ? sums[NB - 2 + k] : sums[k];
        float h, rest;
        split16<false>(s, h, rest);
        pair[k] = low ? rest : h;
      }
      qo = NB == 2 && tq >= 2 ? 0u : pack2<false>(pair[0], pair[1]);
      // (at most 2^100, for queries beyond 2^90: scores that differ at all, by 2^-72 before this
      // factor, then leave one another no probability, with this factor as with the true one,
      // which could leave f32's range)
      const float fr = fminf(a.scale * kLog2e4 * 16777216.f * pow2f(e), 0x1p100f);
#pragma unroll
      for (int k = 0; k < 2; ++k) f[k] = __shfl_sync(0xffffffffu, fr, (2 * tq + k) * 4);
    }
    // The keys that this lane's two rows see: positions below lim (of a selection: places of
    // its list), and those that all rows of the job see.
    int lim[2], all;
    if (a.sel) {
      all = sel_keys(start + divide(job.row0, a.group), a.sel_max);
      lim[0] = lim[1] = all;
    } else {
      all = start + divide(job.row0, a.group) + 1;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        lim[k] = start + divide(job.row0 + min(2 * tq + k, job.rows - 1), a.group) + 1;
    }
    const int most = a.sel ? all : start + divide(job.row0 + job.rows - 1, a.group) + 1;

    // O, and (every row alike) the sums of P d of each block and of P
    float o[NB][2][4], off[NB][4] = {}, sum[4] = {};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int u = 0; u < 2; ++u) o[b][u][0] = o[b][u][1] = o[b][u][2] = o[b][u][3] = 0.f;
    float ref[2] = {0.f, 0.f};
    // V's scales enter times 2^vexp: as they are where the first tile's largest is of ordinary size,
    // else by what takes it to [2^-2, 2^-1).  vexp only falls then, when a scale would reach 2.
    constexpr int kUnset = 99;
    int vexp = kUnset;
    // of the references: not yet set, or beyond kFused, where each step computes its exponents anew
    enum : int { kSet, kFar, kNone };
    int state = kNone;
    uint32_t nans = 0;  // of row 2 tq + k: bit 4 k + b, that it sees a value of block b that is NaN

    // --------------------------------------------------------- the tiles --
    for (; x < seg1; ++x) {
      if (alive && __any_sync(0xffffffffu, !mbar_wait(&full[stage], phase, a.status))) {
        alive = false;
        died[warp] = x - w0;
      }
      const uint8_t* st = ring + stage * C::kRecord;
      const int p0 = (x - job.t0) * kTile;
      const bool tail = p0 + kTile > all;
      const int slices = alive ? min(4, (most - p0 + 15) / 16) : 0;
      // V's scales, those of positions 2 lane and 2 lane + 1 by each lane: where they cannot be
      // taken as they are, they are written anew into the stage.  (2 or more and NaN ones have
      // the exponent's top bit.)
      uint32_t d2[NB], any_d = 0;
      uint32_t* d2_at = reinterpret_cast<uint32_t*>(ring + stage * C::kRecord + kRec.v_scales()) + NB * lane;
      if constexpr (NB == 4) {
        const uint4 w = *reinterpret_cast<const uint4*>(d2_at);
        d2[0] = w.x, d2[1] = w.y, d2[2] = w.z, d2[3] = w.w;
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(d2_at);
        d2[0] = w.x, d2[1] = w.y;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) any_d |= d2[b];
      if (slices > 0 && __any_sync(0xffffffffu, any_d & (vexp == 0 ? 0x40004000u : ~0u))) {
        // Behind the end, or behind what a row sees, P is 0, and 0 times NaN is not: scales behind
        // the end are taken out, and NaN ones are, and the blocks and rows that see those remembered.
        bool anew = p0 + kTile > most;
        if (anew) {
#pragma unroll
          for (int b = 0; b < NB; ++b)
            d2[b] &= (p0 + 2 * lane < most ? 0xffffu : 0u) | (p0 + 2 * lane + 1 < most ? 0xffff0000u : 0u);
        }
        auto largest = [&] {  // its bits
          uint32_t m = 0;
#pragma unroll
          for (int b = 0; b < NB; ++b) m = __vmaxu2(m, d2[b] & 0x7fff7fffu);
          return __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
        };
        uint32_t big = largest();
        if (big > 0x7c00u) {
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const bool bad = ((r ? d2[b] >> 16 : d2[b]) & 0x7fffu) > 0x7c00u;
              if (bad) d2[b] &= r ? 0xffffu : 0xffff0000u;
              for (uint32_t lanes = __ballot_sync(0xffffffffu, bad); lanes; lanes &= lanes - 1) {
                const int place = p0 + 2 * (__ffs(lanes) - 1) + r;
#pragma unroll
                for (int k = 0; k < 2; ++k) nans |= (place < lim[k] ? 1u : 0u) << (4 * k + b);
              }
            }
          big = largest();
          anew = true;
        }
        const int large = big >= 0x400u ? static_cast<int>(big >> 10) - 15 : big ? 7 - __clz(big) : -24;
        int next = vexp;
        if (vexp == kUnset ? large < -4 || large > 0 : large + vexp > 0)
          next = min(max(-2 - large, -15), 15);
        else if (vexp == kUnset)
          next = 0;
        if (next != vexp && vexp != kUnset) {
          const float corr = pow2f(next - vexp);
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              off[b][k] *= corr;
              o[b][0][k] *= corr;
              o[b][1][k] *= corr;
            }
        }
        vexp = next;
        if (anew || vexp != 0) {
          const uint32_t half = vexp > -15 ? (vexp + 15) << 10 : 0x200u;  // 2^vexp
#pragma unroll
          for (int b = 0; b < NB; ++b) d2_at[b] = mul2(d2[b], half << 16 | half);
          fence_proxy_async_shared();  // before the next copy into the stage
          __syncwarp();
        }
      }
      // Two times 16 positions at once: independent chains for the scheduler.
      for (int s = 0; s < slices; s += 2) {
        // of positions 16 s on; 16 positions further lie 256 NB bytes of codes and 32 NB of scales
        const uint8_t* sk = st + k_at + s * (256 * NB);
        const uint8_t* sv = st + v_at + s * (256 * NB);
        const uint8_t* sks = st + ks_at + s * (32 * NB);
        const uint8_t* svs = st + vs_at + s * (32 * NB);
        // ---- S = K q^T
        float y[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t kw[2][NB], kd[2][NB / 2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint8_t* kp = sk + (256 * e + 128 * r) * NB;
            const uint8_t* sp = sks + (32 * e + 16 * r) * NB;
            if constexpr (NB == 4) {
              const uint4 w = *reinterpret_cast<const uint4*>(kp);
              kw[r][0] = w.x, kw[r][1] = w.y, kw[r][2] = w.z, kw[r][3] = w.w;
              const uint2 d = *reinterpret_cast<const uint2*>(sp);
              kd[r][0] = d.x, kd[r][1] = d.y;
            } else {
              const uint2 w = *reinterpret_cast<const uint2*>(kp);
              kw[r][0] = w.x, kw[r][1] = w.y;
              kd[r][0] = *reinterpret_cast<const uint32_t*>(sp);
            }
          }
          const uint32_t* wp = reinterpret_cast<const uint32_t*>(st + kw_at + 32 * (s + e) * NB);
          mma_f16_k8(y[e], wp[0], wp[4 * NB], qo);
#pragma unroll
          for (int k = 0; k < 4; ++k) y[e][k] *= 256.f / 16777216.f;
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            float c[4];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
              const uint32_t u0 = kw[0][b] >> (8 * ks), u1 = kw[1][b] >> (8 * ks);
              const uint32_t a0 = u0 & 0x000f000fu, a1 = u1 & 0x000f000fu;
              const uint32_t a2 = u0 & 0x00f000f0u, a3 = u1 & 0x00f000f0u;
              if (ks == 0)
                mma_f16_first(c, a0, a1, a2, a3, qh[b][0][0], qh[b][0][1]);
              else
                mma_f16(c, a0, a1, a2, a3, qh[b][1][0], qh[b][1][1]);
              if constexpr (LO) mma_f16(c, a0, a1, a2, a3, ql[b][ks][0], ql[b][ks][1]);
            }
            const float d0 = half_of(kd[0][b / 2], b & 1), d1 = half_of(kd[1][b / 2], b & 1);
            y[e][0] = fmaf(c[0], d0, y[e][0]);
            y[e][1] = fmaf(c[1], d0, y[e][1]);
            y[e][2] = fmaf(c[2], d1, y[e][2]);
            y[e][3] = fmaf(c[3], d1, y[e][3]);
          }
        }
        // ---- V's scales of positions 2 tq, 2 tq + 1 and those plus 8
        uint32_t vd[2][2][NB];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint8_t* sp = svs + (32 * e + 16 * r) * NB;
            if constexpr (NB == 4) {
              const uint4 d = *reinterpret_cast<const uint4*>(sp);
              vd[e][r][0] = d.x, vd[e][r][1] = d.y, vd[e][r][2] = d.z, vd[e][r][3] = d.w;
            } else {
              const uint2 d = *reinterpret_cast<const uint2*>(sp);
              vd[e][r][0] = d.x, vd[e][r][1] = d.y;
            }
          }
        // ---- softmax: columns 2 tq, 2 tq + 1 of positions g and g + 8
        if (tail) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (p0 + 16 * (s + e) + g + 8 * (k >> 1) >= lim[k & 1]) y[e][k] = -CUDART_INF_F;
        }
        float p[2][4];
        bool over = false;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            p[e][k] = fmaf(y[e][k], f[k & 1], -ref[k & 1]);
            over |= p[e][k] > kTop;
          }
        if (__any_sync(0xffffffffu, over) || state != kSet) {
          const bool fresh = state == kNone;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            // NaN does not count
            float m = fmaxf(fmaxf(y[0][k] * f[k], y[0][k + 2] * f[k]),
                            fmaxf(y[1][k] * f[k], y[1][k + 2] * f[k]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            float next = ref[k];
            if ((fresh || m - next > kTop) && m > -CUDART_INF_F) next = m - (kTop - kSlack);
            const float corr = fresh ? 0.f : ex2(ref[k] - next);
            ref[k] = next;
            sum[k] *= corr;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              off[b][k] *= corr;
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                o[b][u][k] *= corr;
                o[b][u][k + 2] *= corr;
              }
            }
          }
          state = __any_sync(0xffffffffu, fabsf(ref[0]) > kFused || fabsf(ref[1]) > kFused) ? kFar : kSet;
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int k = 0; k < 4; ++k) p[e][k] = exponent(y[e][k], f[k & 1], ref[k & 1]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int k = 0; k < 4; ++k) p[e][k] = ex2(p[e][k]);
          const uint32_t pt0 = transpose8(pack2<false>(p[e][0], p[e][1]));
          const uint32_t pt1 = transpose8(pack2<false>(p[e][2], p[e][3]));
          // ---- O += V^T (P d), and the sums
          mma_f16(sum, kOnes, kOnes, kOnes, kOnes, pt0, pt1);
          uint32_t vw[2][NB];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint8_t* vp = sv + (256 * e + 128 * r) * NB;
            if constexpr (NB == 4) {
              const uint4 w = *reinterpret_cast<const uint4*>(vp);
              vw[r][0] = w.x, vw[r][1] = w.y, vw[r][2] = w.z, vw[r][3] = w.w;
            } else {
              const uint2 w = *reinterpret_cast<const uint2*>(vp);
              vw[r][0] = w.x, vw[r][1] = w.y;
            }
          }
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint32_t b0 = mul2(pt0, vd[e][0][b]), b1 = mul2(pt1, vd[e][1][b]);
            mma_f16(off[b], kOnes, kOnes, kOnes, kOnes, b0, b1);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t u0 = vw[0][b] >> (8 * u), u1 = vw[1][b] >> (8 * u);
              mma_f16(o[b][u], u0 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x000f000fu,
                      u1 & 0x00f000f0u, b0, b1);
            }
          }
        }
      }
      __syncwarp();  // the stage is free
      if (alive && x + S < w1) issue(x + S - w0, stage);
      if (++stage == S) {
        stage = 0;
        phase ^= 1;
      }
    }

    // ------------------------------------------------- the end of a piece --
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (sum[k] == 0.f) ref[k] = -CUDART_INF_F;  // the row sees none of these tiles
    const bool whole = job.t0 >= w0 && job.t0 + job.tiles <= w1;
    // A piece that ends the warp's part goes into its ring; an earlier one (of a job that
    // other warps began) into memory: the CTA's own piece of it if no other warp here has one.
    float* part = seg1 == w1 ? reinterpret_cast<float*>(ring)
                  : warp == 0 ? a.cta_parts + static_cast<size_t>(2 * blockIdx.x) * C::kPart
                              : a.warp_parts + static_cast<size_t>(blockIdx.x * W + warp) * C::kPart;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = 2 * tq + k;
      const bool live = r < job.rows;
      const float f24 = 16777216.f * pow2f(vexp == kUnset ? 0 : -vexp) * (whole ? 1.f / sum[k] : 1.f);
      const size_t base = whole && live ? row_offset(a, job, job.row0 + r, HD) : 0;
      float eight[NB];  // 8 sum P d of each block, in the units of O
#pragma unroll
      for (int b = 0; b < NB; ++b) eight[b] = off[b][k] * (8.f / 16777216.f);
      if (!live) continue;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float4 v = make_float4((o[b][0][k] - eight[b]) * f24,
                               (o[b][0][k + 2] * 0.0625f - eight[b]) * f24,
                               (o[b][1][k] - eight[b]) * f24,
                               (o[b][1][k + 2] * 0.0625f - eight[b]) * f24);
        if (nans >> (4 * k + b) & 1u) v.x = v.y = v.z = v.w = CUDART_NAN_F;
        const int d = 32 * b + 4 * g;
        if (whole)
          store4(a.out, base + d, a.out_dtype, v, a.out_vec != 0);
        else
          *reinterpret_cast<float4*>(part + r * HD + d) = v;
      }
      if (!whole && g == 0) *reinterpret_cast<float2*>(part + 8 * HD + 2 * r) = make_float2(ref[k], sum[k]);
    }
  }

  // (the status says so; the warp's other copies in flight are waited for, as long again)
  if (!alive) {
#pragma unroll 1
    for (int i = died[warp], n = min(i + S, w1 - w0); i < n; ++i)
      mbar_wait(&full[i % S], i / S & 1, a.status);
  }
  if (lane == 0 && w0 < w1) last_job[warp] = job;

  // ------------------------------------------------------------ joining --
  // (__syncthreads orders the pieces in memory as well, inside the CTA)
  __syncthreads();
  // The first job of the run, if another CTA began it and it ends in the first warp's part; then
  // the last job of each warp's part, where its first tile here lies.  (Loops that are not
  // unrolled: every launch runs this code cold.)
  auto warp_begin = [&](int i) { return min(c0 + i * a.per_warp, c1); };
  // Sums the n pieces part(0) .. of job j into the output, or into the piece `into`.
  auto join = [&](const Job& j, int n, float* into, auto part) {
#pragma unroll 1
    for (int c = threadIdx.x; c < j.rows * (HD / 4); c += 32 * W) {
      const int r = c / (HD / 4), d = c % (HD / 4) * 4;
      float ref = -CUDART_INF_F, sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const float* p = part(k);
        const float2 ml = *reinterpret_cast<const float2*>(p + 8 * HD + 2 * r);
        const float4 v = *reinterpret_cast<const float4*>(p + r * HD + d);
        const float most = fmaxf(ref, ml.x), base = most == -CUDART_INF_F ? 0.f : most;
        const float f0 = ex2(ref - base), f1 = ex2(ml.x - base);
        sum = sum * f0 + ml.y * f1;
        acc.x = acc.x * f0 + v.x * f1;
        acc.y = acc.y * f0 + v.y * f1;
        acc.z = acc.z * f0 + v.z * f1;
        acc.w = acc.w * f0 + v.w * f1;
        ref = most;
      }
      if (into) {
        *reinterpret_cast<float4*>(into + r * HD + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(into + 8 * HD + 2 * r) = make_float2(ref, sum);
      } else {
        const float f = 1.f / sum;
        store4(a.out, row_offset(a, j, j.row0 + r, HD) + d, a.out_dtype,
               make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f), a.out_vec != 0);
      }
    }
  };
  Job open[2];  // jobs that other CTAs have pieces of: the run's first and its last
  int opens = 0;
  if (c0 < c1 && last_job[0].t0 > c0) {  // (its piece is in the CTA's place already)
    open[0] = job_at(a, c0);
    opens = open[0].t0 < c0;
  }
#pragma unroll 1
  for (int i = 0; i < W; ++i) {
    const int b0 = warp_begin(i), b1 = warp_begin(i + 1);
    if (b0 >= b1) break;
    const Job j = last_job[i];
    const int t1 = j.t0 + j.tiles, end = min(t1, c1);
    if ((j.t0 >= b0 && t1 <= b1) || (j.t0 < b0 && i > 0)) continue;
    int n = 1;
    while (i + n < W && warp_begin(i + n) < end) ++n;
    const bool inside = j.t0 >= c0 && t1 <= c1;
    join(j, n,
         inside ? nullptr
                : a.cta_parts + static_cast<size_t>(2 * blockIdx.x + (j.t0 > c0 ? 1 : 0)) * C::kPart,
         [&](int k) -> const float* {
           return end >= warp_begin(i + k + 1)
                      ? reinterpret_cast<const float*>(smem + (i + k) * ring_bytes)
                      : a.warp_parts + static_cast<size_t>(blockIdx.x * W + i + k) * C::kPart;
         });
    if (!inside) open[opens++] = j;
  }
  if (opens == 0) return;
  // The barrier orders every thread's part of the pieces before the counts, whose release makes
  // them visible; the last CTA's acquire sees the others'.
  __syncthreads();
  if (lane == 0 && warp < opens) {
    const Job j = open[warp];
    const int others = divide(j.t0 + j.tiles - 1, a.per_cta) - divide(j.t0, a.per_cta);
    flag[warp] = atom_add_acq_rel_gpu(&a.counters[j.id], 1) == others;
    if (flag[warp]) a.counters[j.id] = 0;
  }
  __syncthreads();
#pragma unroll 1
  for (int o = 0; o < opens; ++o) {
    if (!flag[o]) continue;
    const Job j = open[o];
    const int first = divide(j.t0, a.per_cta), last = divide(j.t0 + j.tiles - 1, a.per_cta);
    join(j, last - first + 1, nullptr, [&](int k) -> const float* {
      const int c = first + k;
      return a.cta_parts + static_cast<size_t>(2 * c + (j.t0 > c * a.per_cta ? 1 : 0)) * C::kPart;
    });
  }
}

bool attn4_supported(int hd, int page) { return (hd == 64 || hd == 128) && page % kTile == 0; }

namespace {

template <int HD, bool LO>
cudaError_t launch_attn4_t(const Attn4Args& a, cudaStream_t s) {
  using C = Attn4Cfg<HD>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = ql_once_per_device(done, [] {
    return cudaFuncSetAttribute(attn4_kernel<HD, LO>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(C::smem(C::kStages)));
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.total + a.per_cta - 1) / a.per_cta);
  cfg.blockDim = dim3(32 * C::kWarps);
  cfg.dynamicSmemBytes = C::smem(a.stages);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attn4_kernel<HD, LO>, a);
}

}  // namespace

// The split of the tiles (tiles[b] of each of sequence b's `jobs` jobs) over CTAs and warps.
// Each CTA takes an equal run of the list (one CTA an SM: a warp's ring fills its share of the
// shared memory).  Where as many CTAs as there are SMs can be given whole shares of jobs with no
// warp taking longer than in an equal split, the list is padded so that a CTA's run stays inside
// one job: one piece a CTA to join instead of two.
int attn4_plan(int hd, int num_sms, const int* tiles, int batch, int jobs, Attn4Args* a,
               size_t* cta_bytes, size_t* warp_bytes) {
  constexpr int kMinTiles = 4;  // of a CTA: fewer cost more in joining than they save
  const int warps = hd == 128 ? Attn4Cfg<128>::kWarps : Attn4Cfg<64>::kWarps;
  const int part = hd == 128 ? Attn4Cfg<128>::kPart : Attn4Cfg<64>::kPart;
  const int most_stages = hd == 128 ? Attn4Cfg<128>::kStages : Attn4Cfg<64>::kStages;
  int64_t total = 0;
  int longest = 1;
  for (int b = 0; b < batch; ++b) {
    total += static_cast<int64_t>(tiles[b]) * jobs;
    longest = std::max(longest, tiles[b]);
  }
  // (what the kernel's divide() takes; padding below adds no more than a share of each job)
  if (total > (1 << 30) || jobs >= (1 << 22)) return 1;
  const int ctas = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(num_sms, (total + kMinTiles - 1) / kMinTiles)));
  a->per_cta = static_cast<int>((total + ctas - 1) / ctas);
  a->aligned = 0;
  const int per_warp = (a->per_cta + warps - 1) / warps;
  // the smallest share of a job that leaves no more CTAs than SMs (the longest sequence's alone
  // may not be more)
  const bool room = static_cast<int64_t>(batch) * jobs <= num_sms;
  for (int splits = room ? std::min(longest, num_sms / jobs) : 0; splits >= 1; --splits) {
    const int share = std::max((longest + splits - 1) / splits, std::min(longest, kMinTiles));
    int64_t n = 0;
    for (int b = 0; b < batch; ++b) n += static_cast<int64_t>((tiles[b] + share - 1) / share) * jobs;
    if (n > num_sms) continue;
    if ((share + warps - 1) / warps <= per_warp) {
      a->per_cta = share;
      a->aligned = 1;
    }
    break;
  }
  a->per_warp = (a->per_cta + warps - 1) / warps;
  a->stages = std::min(most_stages, a->per_warp);
  total = 0;
  for (int b = 0; b < batch; ++b) {
    a->first[b] = static_cast<int32_t>(total);
    const int t = a->aligned ? (tiles[b] + a->per_cta - 1) / a->per_cta * a->per_cta : tiles[b];
    total += static_cast<int64_t>(t) * jobs;
  }
  a->total = static_cast<int32_t>(total);
  const size_t n = static_cast<size_t>((total + a->per_cta - 1) / a->per_cta);
  *cta_bytes = n * 2 * part * sizeof(float);
  *warp_bytes = n * warps * part * sizeof(float);
  return 0;
}

cudaError_t launch_attn4(const Attn4Args& a, cudaStream_t s) {
  const bool lo = a.in_dtype == kF32 || a.rope_stride != 0;
  if (a.cache.hd == 128)
    return lo ? launch_attn4_t<128, true>(a, s) : launch_attn4_t<128, false>(a, s);
  return lo ? launch_attn4_t<64, true>(a, s) : launch_attn4_t<64, false>(a, s);
}

}  // namespace ql
