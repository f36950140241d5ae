// verify.cu -- verification of drafted tokens (speculative decoding).
//
// vtq_verify_draft. Draft i of a sequence, token x_i drawn from q_i, is kept
// while u_i < p_i(x_i) / q_i(x_i), tested as u_i q_i(x_i) < p_i(x_i) in 64 bits
// (the product of two 32-bit numbers is exact there). At the first rejection a
// token is drawn from r = max(p - q, 0) / sum, after the last draft from
// r = p / sum: the lowest v with r_0 + .. + r_v > u_K (r_0 + .. + r_{V-1}).
// This keeps the target's distribution whatever the draft's was.
//
// vtq_verify_greedy. Draft i is kept while it is the lowest index of the
// largest logit of row i; the token behind is the next row's.
//
// What bounds them: one row of p and one of q for each sequence (the row of
// the first rejection), read once. One cluster works on one sequence, so that
// a single sequence still reads with up to 8 SMs and no workspace or second
// launch is needed. A lane's sums are a 32-bit value and its rounding errors
// (together about 48 bits), everything above a lane is in 64 bits, in an order
// that V and the cluster size alone decide: plain 32-bit sums move the cut
// between two tokens by about 1e-7 of the total, which over 1e5 tokens is a
// different token once in some hundred draws. 128 x 8 rows of 100003 in f32,
// two thirds of the sequences with a rejection: 27 us for 85 MB (3.2 TB/s,
// floor 13 us: the error sums take instructions, the ends of the pass latency).
// Greedy, 64 x 8 rows of 32000 in f32, 3.2 rows a sequence needed (26 MB, 4 us):
// 16 us for the 34 MB that groups of four rows read, 23 with single values a
// load. Not HBM bounds it but two groups in a chain, each its load, its
// reduction and a cluster barrier.
#include <cooperative_groups.h>

#include <algorithm>

#include "serve.h"
#include "tc5.cuh"

namespace cg = cooperative_groups;

namespace vtq {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;  // four CTAs an SM
constexpr int kStrips = 8, kBlock = 32 * kStrips;  // elements summed by one warp at a time
static_assert(kWarps >= 4 && kWarps <= 32, "the joins below take one warp a row and one lane a warp");

struct VerifyParams {
  const int32_t* draft;
  int64_t ld_draft;
  const int32_t* n_draft;  // may be null: K for all
  const void* p;
  int64_t p_seq, p_row;
  const void* q;  // may be null: each draft was its only choice
  int64_t q_seq, q_row;
  const float* u;
  int64_t ld_u;
  int K;
  int64_t V;
  int32_t* tokens;
  int64_t ld_tokens;
  int32_t* accepted;
};

__device__ __forceinline__ int draft_count(const VerifyParams& a, int b) {
  return a.n_draft ? min(max(a.n_draft[b], 0), a.K) : a.K;
}

// What is left of p at one token after q: r of the header comment, as its 32-bit value and that
// value's own rounding error (together exact). NaN counts as nothing. A conversion of each value to 64
// bits instead takes the conversion unit's whole time: 109 us where this form takes a quarter of it
// (128 rows of 100003 tokens).
struct Left {
  float r, e;
};
template <typename T>
__device__ __forceinline__ Left left(float p, float q) {
  Left w;
  w.r = __fsub_rn(p, q);
  if (!(w.r > 0.0f)) return Left{0.0f, 0.0f};
  const float t = __fsub_rn(w.r, p);
  w.e = __fsub_rn(__fsub_rn(p, __fsub_rn(w.r, t)), __fadd_rn(q, t));
  return w;
}
// The kStrips values of both rows at e0, e0 + 32, ..: nothing behind v1.
template <typename T>
struct Strips {
  T a[kStrips], b[kStrips];
  __device__ __forceinline__ void load(const T* p, const T* q, int64_t e0, int64_t v1, bool sub) {
    const int n = (int)min(v1 - e0, (int64_t)kBlock);  // of this lane's places
    const T *pe = p + e0, *qe = sub && q ? q + e0 : nullptr;
    if (__all_sync(0xffffffffu, n > 32 * (kStrips - 1))) {
#pragma unroll
      for (int k = 0; k < kStrips; k++) {
        a[k] = pe[32 * k];
        b[k] = qe ? qe[32 * k] : from_f32<T>(0.0f);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kStrips; k++) {
        a[k] = 32 * k < n ? pe[32 * k] : from_f32<T>(0.0f);
        b[k] = 32 * k < n && qe ? qe[32 * k] : from_f32<T>(0.0f);
      }
    }
  }
  __device__ __forceinline__ Left left_at(int k, int64_t e0, int64_t only, bool sub) const {
    return left<T>(to_f32(a[k]), sub && e0 + 32 * k == only ? 1.0f : to_f32(b[k]));
  }
};

__device__ __forceinline__ double warp_sum(double s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
__device__ __forceinline__ double warp_scan(double s, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  return s;
}

// One cluster a sequence. CTA c of the cluster owns the blocks of kBlock
// tokens [c nb, (c + 1) nb).
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) verify_draft_kernel(const VerifyParams a, int nb) {
  extern __shared__ double sums[];  // nb: block sums, then their inclusive scan
  __shared__ int s_acc;
  __shared__ double s_total, s_warp[kWarps];
  __shared__ int64_t s_last, s_lastw[kWarps];
  tc5::grid_wait();
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), size = (int)cl.num_blocks();
  const int b = blockIdx.x / size;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* P = static_cast<const T*>(a.p) + (int64_t)b * a.p_seq;
  const T* Q = a.q ? static_cast<const T*>(a.q) + (int64_t)b * a.q_seq : nullptr;
  const int32_t* draft = a.draft + (int64_t)b * a.ld_draft;
  const float* u = a.u + (int64_t)b * a.ld_u;
  const int n = draft_count(a, b);
  if (warp == 0) {
    int acc = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      bool keep = false;
      if (i < n) {
        const int64_t x = draft[i];
        if (x >= 0 && x < a.V) {
          const double px = to_f32(P[i * a.p_row + x]);
          const double qx = Q ? to_f32(Q[i * a.q_row + x]) : 1.0f;
          keep = (double)u[i] * qx < px;
        }
      }
      const unsigned gone = ~__ballot_sync(0xffffffffu, keep);
      if (gone) {
        acc = i0 + __ffs(gone) - 1;
        break;
      }
      acc = i0 + 32;
    }
    if (lane == 0) s_acc = min(acc, n);
  }
  __syncthreads();
  const int acc = s_acc;
  const T* p = P + acc * a.p_row;
  const T* q = Q && acc < n ? Q + acc * a.q_row : nullptr;
  const int64_t only = acc < n && !Q ? (int64_t)draft[acc] : -1;
  const int64_t v0 = (int64_t)rank * nb * kBlock, v1 = min(a.V, v0 + (int64_t)nb * kBlock);
  const int mine = v1 > v0 ? (int)((v1 - v0 + kBlock - 1) / kBlock) : 0;

  // Twice at most: where p - q leaves nothing at all, the token is drawn from p.
  for (int pass = 0; pass < 2; pass++) {
    const bool sub = pass == 0 && acc < n;
    for (int j = warp; j < mine; j += kWarps) {
      const int64_t e0 = v0 + (int64_t)j * kBlock + lane;
      Strips<T> now;
      now.load(p, q, e0, v1, sub);
      // This lane's sum as a 32-bit value and what its roundings lost: 2^-48 of it.
      float hi = 0.0f, lo = 0.0f;
#pragma unroll
      for (int k = 0; k < kStrips; k++) {
        const Left r = now.left_at(k, e0, only, sub);
        const float s = __fadd_rn(hi, r.r), t = __fsub_rn(s, hi);
        lo = __fadd_rn(lo, __fadd_rn(__fadd_rn(__fsub_rn(hi, __fsub_rn(s, t)), __fsub_rn(r.r, t)), r.e));
        hi = s;
      }
      const double s = warp_sum((double)hi + (double)lo);
      if (lane == 0) sums[j] = s;
    }
    __syncthreads();
    // Inclusive scan of the block sums: each thread a run of them, then the runs.
    const int per = (mine + kThreads - 1) / kThreads, j0 = min(tid * per, mine), j1 = min(j0 + per, mine);
    double s = 0.0;
    for (int j = j0; j < j1; j++) {
      s += sums[j];
      sums[j] = s;
    }
    const double inc = warp_scan(s, lane);
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    double base = __shfl_up_sync(0xffffffffu, inc, 1);
    if (lane == 0) base = 0.0;
    double before = 0.0;
    for (int w = 0; w < warp; w++) before += s_warp[w];
    base += before;
    for (int j = j0; j < j1; j++) sums[j] += base;
    __syncthreads();
    if (tid == 0) s_total = mine ? sums[mine - 1] : 0.0;
    cl.sync();
    // The other CTAs' totals, in rank order: the same numbers in every CTA.
    double total = 0.0, start = 0.0;
    for (int c = 0; c < size; c++) {
      if (c == rank) start = total;
      total += *cl.map_shared_rank(&s_total, c);
    }
    if (pass == 0 && sub && !(total > 0.0)) {
      cl.sync();  // everybody has read the totals; the next pass writes them again
      continue;
    }
    const double cut = fmax((double)u[a.K] * total, 0.0);
    int64_t any = -1;
    if (!(total > cut)) {
      // u of 1 or more, or no finite total: the last token that has any weight.
      int64_t last = -1;
      for (int j = warp; j < mine; j += kWarps) {
        const int64_t e0 = v0 + (int64_t)j * kBlock + lane;
        Strips<T> now;
        now.load(p, q, e0, v1, sub);
#pragma unroll
        for (int k = 0; k < kStrips; k++)
          if (now.left_at(k, e0, only, sub).r > 0.0f) last = e0 + 32 * k;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        const int64_t t = __shfl_xor_sync(0xffffffffu, last, o);
        last = last > t ? last : t;
      }
      if (lane == 0) s_lastw[warp] = last;
      __syncthreads();
      if (tid == 0) {
        int64_t l = -1;
        for (int w = 0; w < kWarps; w++) l = l > s_lastw[w] ? l : s_lastw[w];
        s_last = l;
      }
      cl.sync();
      for (int c = 0; c < size; c++) {
        const int64_t l = *cl.map_shared_rank(&s_last, c);
        any = any > l ? any : l;
      }
    }
    const double end = start + s_total;  // the sum that the next CTA takes for its start
    int32_t* out = a.tokens + (int64_t)b * a.ld_tokens;
    if (rank == 0) {
      for (int i = tid; i <= a.K; i += kThreads)
        if (i != acc) out[i] = i < acc ? draft[i] : -1;
      if (tid == 0) {
        a.accepted[b] = acc;
        if (!(total > cut)) out[acc] = (int32_t)any;
      }
    }
    if (total > cut && !(start > cut) && end > cut) {
      // The cut lies in this CTA: its block, then the token, by warp 0.
      if (warp == 0) {
        int lo = 0, hi = mine - 1;
        while (lo < hi) {
          const int m = (lo + hi) >> 1;
          if (start + sums[m] > cut) hi = m;
          else lo = m + 1;
        }
        // The block's sum passed the cut; its scan, rounded in another order, may just not: then the
        // block's last token with any weight (or, where the block has none, of one before it).
        int64_t found = -1, tail = -1;
        for (int j = lo; j >= 0 && tail < 0; j--) {
          double cum = j ? sums[j - 1] : 0.0;
          const int64_t e0 = v0 + (int64_t)j * kBlock + lane;
          Strips<T> now;
          now.load(p, q, e0, v1, sub);
#pragma unroll
          for (int k = 0; k < kStrips; k++) {
            const Left r = now.left_at(k, e0, only, sub);
            const double c = warp_scan((double)r.r + (double)r.e, lane);
            const unsigned over = __ballot_sync(0xffffffffu, r.r > 0.0f && start + (cum + c) > cut);
            const unsigned some = __ballot_sync(0xffffffffu, r.r > 0.0f);
            if (found < 0 && over) found = e0 - lane + 32 * k + __ffs(over) - 1;
            if (some) tail = e0 - lane + 32 * k + 31 - __clz(some);
            cum += __shfl_sync(0xffffffffu, c, 31);
          }
        }
        if (lane == 0) out[acc] = (int32_t)(found >= 0 ? found : tail);
      }
    }
    cl.sync();  // no CTA leaves while another still reads its total
    return;
  }
}

// A row's argmax as the larger of 64-bit keys: the value's bits, put in the order of the values, above
// the complement of the index, so that the lower index wins a tie. NaN is never larger (key 0), and a
// NaN at index 0 is never passed (the order of the decode loop's own argmax).
__device__ __forceinline__ void take(float x, uint32_t v, uint32_t& hi, uint32_t& lo) {
  const uint32_t bits = __float_as_uint(__fadd_rn(x, 0.0f));  // -0 is 0
  uint32_t k = bits ^ ((int32_t)bits < 0 ? 0xffffffffu : 0x80000000u);
  if (x != x) k = v == 0 ? 0xffffffffu : 0u;
  const uint32_t i = ~v;
  if (k > hi || (k == hi && i > lo)) hi = k, lo = i;
}

constexpr int kGroup = 4;  // rows looked at together: a chain of drafts waits for two groups, not eight rows

// VEC: rows of whole 16-byte pieces.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) verify_greedy_kernel(const VerifyParams a) {
  __shared__ uint2 s_warp[kGroup][kWarps];
  __shared__ uint2 s_key[2][kGroup];  // two sets: a CTA may be one group ahead of another's reads
  tc5::grid_wait();
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), size = (int)cl.num_blocks();
  const int b = blockIdx.x / size;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* P = static_cast<const T*>(a.p) + (int64_t)b * a.p_seq;
  const int32_t* draft = a.draft + (int64_t)b * a.ld_draft;
  int32_t* out = a.tokens + (int64_t)b * a.ld_tokens;
  const int n = draft_count(a, b);
  const uint32_t V = (uint32_t)a.V, step = (uint32_t)(size * kThreads);
  int acc = 0;
  int32_t token = 0;
  for (int set = 0;; set ^= 1) {
    const int rows = min(kGroup, n + 1 - acc);
    uint32_t hi[kGroup], lo[kGroup];
#pragma unroll
    for (int r = 0; r < kGroup; r++) hi[r] = lo[r] = 0;
    const T* p = P + acc * a.p_row;
    if constexpr (VEC) {
      constexpr uint32_t W = 16 / sizeof(T);
      const uint32_t chunks = V / W;
      for (uint32_t c0 = (uint32_t)(rank * kThreads + tid); c0 < chunks; c0 += step * 2) {
        uint4 x[kGroup][2];
#pragma unroll
        for (int r = 0; r < kGroup; r++)
#pragma unroll
          for (int k = 0; k < 2; k++)
            if (r < rows && c0 + k * step < chunks) x[r][k] = reinterpret_cast<const uint4*>(p + r * a.p_row)[c0 + k * step];
#pragma unroll
        for (int r = 0; r < kGroup; r++)
#pragma unroll
          for (int k = 0; k < 2; k++) {
            if (r >= rows || c0 + k * step >= chunks) continue;
            const T* e = reinterpret_cast<const T*>(&x[r][k]);
#pragma unroll
            for (uint32_t i = 0; i < W; i++) take(to_f32(e[i]), (c0 + k * step) * W + i, hi[r], lo[r]);
          }
      }
    } else {
      for (uint32_t v0 = (uint32_t)(rank * kThreads + tid); v0 < V; v0 += step * 4) {
        float x[kGroup][4];
#pragma unroll
        for (int r = 0; r < kGroup; r++)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const uint32_t v = v0 + k * step;
            x[r][k] = r < rows && v < V ? to_f32(p[r * a.p_row + v]) : __uint_as_float(0x7fc00000u);
          }
#pragma unroll
        for (int r = 0; r < kGroup; r++)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const uint32_t v = v0 + k * step;
            if (v < V) take(x[r][k], v, hi[r], lo[r]);
          }
      }
    }
#pragma unroll
    for (int r = 0; r < kGroup; r++) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, hi[r]);
      const uint32_t i = __reduce_max_sync(0xffffffffu, hi[r] == m ? lo[r] : 0u);
      if (lane == 0) s_warp[r][warp] = make_uint2(m, i);
    }
    __syncthreads();
    if (warp < kGroup) {
      const uint2 k = lane < kWarps ? s_warp[warp][lane] : make_uint2(0, 0);
      const uint32_t m = __reduce_max_sync(0xffffffffu, k.x);
      const uint32_t i = __reduce_max_sync(0xffffffffu, k.x == m ? k.y : 0u);
      if (lane == 0) s_key[set][warp] = make_uint2(m, i);
    }
    cl.sync();
    // Every warp of every CTA joins the same keys: lane = (CTA, row).
    uint2 k = make_uint2(0, 0);
    if (lane < size * kGroup) k = cl.map_shared_rank(&s_key[set][0], lane / kGroup)[lane % kGroup];
#pragma unroll
    for (int o = kGroup; o < 32; o <<= 1) {
      const uint32_t oh = __shfl_xor_sync(0xffffffffu, k.x, o), ol = __shfl_xor_sync(0xffffffffu, k.y, o);
      if (oh > k.x || (oh == k.x && ol > k.y)) k = make_uint2(oh, ol);
    }
    const int32_t best = k.x ? (int32_t)~k.y : 0;  // of row acc + lane % kGroup; nothing but NaN: 0
    const int r = lane % kGroup;
    const bool keep = r < rows && acc + r < n && draft[acc + r] == best;
    const unsigned gone = ~__ballot_sync(0xffffffffu, keep) & ((1u << kGroup) - 1);
    if (gone) {
      const int first = __ffs(gone) - 1;
      acc += first;
      token = __shfl_sync(0xffffffffu, best, first);
      break;
    }
    acc += kGroup;
  }
  if (rank == 0) {
    for (int i = tid; i <= a.K; i += kThreads) out[i] = i < acc ? draft[i] : i == acc ? token : -1;
    if (tid == 0) a.accepted[b] = acc;
  }
  cl.sync();  // no CTA leaves while another still reads its keys
}

// CTAs a sequence: enough that every SM holds a few, each with some thousand tokens of its own.
int cluster_size(int64_t seqs, int64_t V) {
  int c = 1;
  while (c < 8 && seqs * c < 3 * num_sms() && V > (int64_t)c * 2048) c *= 2;
  return c;
}

template <typename T>
cudaError_t launch_draft(const VerifyParams& p, int64_t seqs, int cluster, int nb, cudaStream_t st) {
  static std::atomic<uint64_t> allowed{0};
  const size_t smem = (size_t)nb * sizeof(double);
  if (smem > 48 * 1024 - 1024) {
    const cudaError_t e = allow_smem((const void*)verify_draft_kernel<T>, smem, allowed);
    if (e != cudaSuccess) return e;
  }
  return launch_after(verify_draft_kernel<T>, dim3((unsigned)(seqs * cluster)), kThreads, smem, cluster, st, p, nb);
}

template <typename T>
cudaError_t launch_greedy(const VerifyParams& p, int64_t seqs, int cluster, cudaStream_t st) {
  constexpr int64_t W = 16 / sizeof(T);
  const dim3 grid((unsigned)(seqs * cluster));
  if (aligned16(p.p) && p.V % W == 0 && p.p_row % W == 0 && p.p_seq % W == 0)
    return launch_after(verify_greedy_kernel<T, true>, grid, kThreads, 0, cluster, st, p);
  return launch_after(verify_greedy_kernel<T, false>, grid, kThreads, 0, cluster, st, p);
}

vtq_status check(const char* fn, const vtq_verify_args* a, bool greedy) {
  if (!a) return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null arguments", fn);
  if (!serve_elt(a->dtype))
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (rows not F32 / F16 / BF16)", fn);
  if (a->seqs < 0 || a->drafts < 0 || a->vocab < 1)
    return serve_fail(VTQ_ERR_INTERNAL, "%s: bad shape", fn);
  // 8 CTAs at most hold a row's block sums in 200 KB of shared memory each.
  if (a->vocab > (1 << 24) || a->drafts > (1 << 16) || a->seqs > (1 << 24))
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED,
                      "%s: not implemented (vocab or seqs over 2^24, drafts over 2^16)", fn);
  if (a->seqs == 0) return VTQ_OK;
  if ((!a->draft && a->drafts) || !a->target || (!greedy && !a->u) || !a->tokens || !a->accepted)
    return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null pointer", fn);
  return VTQ_OK;
}

VerifyParams params(const vtq_verify_args* a) {
  return VerifyParams{a->draft,      a->ld_draft,   a->n_draft,    a->target,      a->target_seq,
                      a->target_row, a->proposal,   a->proposal_seq, a->proposal_row, a->u,
                      a->ld_u,       (int)a->drafts, a->vocab,     a->tokens,      a->ld_tokens,
                      a->accepted};
}

}  // namespace
}  // namespace vtq

using namespace vtq;

extern "C" {

vtq_status vtq_verify_draft(const vtq_verify_args* a, void* stream) {
  if (vtq_status s = check("vtq_verify_draft", a, false)) return s;
  if (a->seqs == 0) return VTQ_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int c = cluster_size(a->seqs, a->vocab);
  const int64_t blocks = (a->vocab + kBlock - 1) / kBlock;
  const int nb = (int)((blocks + c - 1) / c);
  const VerifyParams p = params(a);
  if ((size_t)nb * sizeof(double) > 200 * 1024)
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "vtq_verify_draft: not implemented (vocab too large)");
  const cudaError_t e = a->dtype == VTQ_F32   ? launch_draft<float>(p, a->seqs, c, nb, st)
                        : a->dtype == VTQ_F16 ? launch_draft<__half>(p, a->seqs, c, nb, st)
                                              : launch_draft<__nv_bfloat16>(p, a->seqs, c, nb, st);
  return serve_cuda(e, "vtq_verify_draft");
}

vtq_status vtq_verify_greedy(const vtq_verify_args* a, void* stream) {
  if (vtq_status s = check("vtq_verify_greedy", a, true)) return s;
  if (a->seqs == 0) return VTQ_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int c = cluster_size(a->seqs, a->vocab);
  const VerifyParams p = params(a);
  const cudaError_t e = a->dtype == VTQ_F32   ? launch_greedy<float>(p, a->seqs, c, st)
                        : a->dtype == VTQ_F16 ? launch_greedy<__half>(p, a->seqs, c, st)
                                              : launch_greedy<__nv_bfloat16>(p, a->seqs, c, st);
  return serve_cuda(e, "vtq_verify_greedy");
}

}  // extern "C"
