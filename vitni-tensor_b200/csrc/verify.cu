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
// launch is needed. Sums are in 64 bits in an order that V and the cluster
// size alone decide: 32-bit sums move the cut between two tokens by about
// 1e-7 of the total, which over 1e5 tokens is a different token once in some
// hundred draws.
#include <cooperative_groups.h>

#include <algorithm>

#include "serve.h"
#include "vtq_internal.h"

namespace cg = cooperative_groups;

namespace vtq {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kStrips = 8, kBlock = 32 * kStrips;  // elements summed by one warp at a time

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

// What is left of p at one token after q: r of the header comment. NaN counts as nothing.
template <typename T>
__device__ __forceinline__ double left(const T* p, const T* q, int64_t v, int64_t only, bool sub) {
  double r = (double)to_f32(p[v]);
  if (sub) r -= q ? (double)to_f32(q[v]) : (v == only ? 1.0 : 0.0);
  return r > 0.0 ? r : 0.0;
}

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
__global__ void __launch_bounds__(kThreads) verify_draft_kernel(const VerifyParams a, int nb) {
  extern __shared__ double sums[];  // nb: block sums, then their inclusive scan
  __shared__ int s_acc;
  __shared__ double s_total, s_warp[kWarps];
  __shared__ int64_t s_last, s_lastw[kWarps];
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
    int64_t last = -1;  // the last token that has any weight
    for (int j = warp; j < mine; j += kWarps) {
      const int64_t e0 = v0 + (int64_t)j * kBlock + lane;
      double r[kStrips];
#pragma unroll
      for (int k = 0; k < kStrips; k++) r[k] = e0 + 32 * k < v1 ? left(p, q, e0 + 32 * k, only, sub) : 0.0;
      double s = 0.0;
#pragma unroll
      for (int k = 0; k < kStrips; k++) {
        s += r[k];
        if (r[k] > 0.0) last = e0 + 32 * k;
      }
      s = warp_sum(s);
      if (lane == 0) sums[j] = s;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const int64_t t = __shfl_xor_sync(0xffffffffu, last, o);
      last = last > t ? last : t;
    }
    if (lane == 0) s_lastw[warp] = last;
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
    if (tid == 0) {
      int64_t l = -1;
      for (int w = 0; w < kWarps; w++) l = l > s_lastw[w] ? l : s_lastw[w];
      s_last = l;
    }
    __syncthreads();
    if (tid == 0) s_total = mine ? sums[mine - 1] : 0.0;
    cl.sync();
    // The other CTAs' totals, in rank order: the same numbers in every CTA.
    double total = 0.0, start = 0.0;
    int64_t any = -1;
    for (int c = 0; c < size; c++) {
      if (c == rank) start = total;
      total += *cl.map_shared_rank(&s_total, c);
      const int64_t l = *cl.map_shared_rank(&s_last, c);
      any = any > l ? any : l;
    }
    if (pass == 0 && sub && !(total > 0.0)) {
      cl.sync();  // everybody has read the totals; the next pass writes them again
      continue;
    }
    const double cut = fmax((double)u[a.K] * total, 0.0);
    const double end = start + s_total;  // the sum that the next CTA takes for its start
    int32_t* out = a.tokens + (int64_t)b * a.ld_tokens;
    if (rank == 0) {
      for (int i = tid; i <= a.K; i += kThreads)
        if (i != acc) out[i] = i < acc ? draft[i] : -1;
      if (tid == 0) {
        a.accepted[b] = acc;
        if (!(total > cut)) out[acc] = (int32_t)any;  // u of 1 or more, or no finite total
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
          double r[kStrips];
#pragma unroll
          for (int k = 0; k < kStrips; k++) r[k] = e0 + 32 * k < v1 ? left(p, q, e0 + 32 * k, only, sub) : 0.0;
#pragma unroll
          for (int k = 0; k < kStrips; k++) {
            const double c = warp_scan(r[k], lane);
            const unsigned over = __ballot_sync(0xffffffffu, r[k] > 0.0 && start + (cum + c) > cut);
            const unsigned some = __ballot_sync(0xffffffffu, r[k] > 0.0);
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

// The order of a row's argmax: larger first, then the lower index. NaN is never larger, and a NaN at
// index 0 is never passed (the order of the decode loop's own argmax).
__device__ __forceinline__ bool better(float v, int64_t i, float best, int64_t at) {
  return v > best || (v == best && i < at);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_greedy_kernel(const VerifyParams a) {
  __shared__ float s_v[2][kWarps];
  __shared__ int64_t s_i[2][kWarps];
  __shared__ float s_best[2];
  __shared__ int64_t s_at[2];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), size = (int)cl.num_blocks();
  const int b = blockIdx.x / size;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* P = static_cast<const T*>(a.p) + (int64_t)b * a.p_seq;
  const int32_t* draft = a.draft + (int64_t)b * a.ld_draft;
  int32_t* out = a.tokens + (int64_t)b * a.ld_tokens;
  const int n = draft_count(a, b);
  int acc = 0;
  int32_t token = 0;
  for (;; acc++) {
    const T* p = P + acc * a.p_row;
    float best = -INFINITY;
    int64_t at = INT64_MAX;
    for (int64_t v0 = (int64_t)rank * kThreads + tid; v0 < a.V; v0 += (int64_t)size * kThreads * 8) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int64_t v = v0 + (int64_t)k * size * kThreads;
        x[k] = v < a.V ? to_f32(p[v]) : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int64_t v = v0 + (int64_t)k * size * kThreads;
        if (v < a.V && better(x[k], v, best, at)) best = x[k], at = v;
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, best, o);
      const int64_t oi = __shfl_xor_sync(0xffffffffu, at, o);
      if (better(ov, oi, best, at)) best = ov, at = oi;
    }
    const int s = acc & 1;  // two sets: a CTA may be one row ahead of another's reads
    if (lane == 0) s_v[s][warp] = best, s_i[s][warp] = at;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWarps; w++)
        if (better(s_v[s][w], s_i[s][w], best, at)) best = s_v[s][w], at = s_i[s][w];
      s_best[s] = best;
      s_at[s] = at;
    }
    cl.sync();
    for (int c = 0; c < size; c++) {
      const float ov = *cl.map_shared_rank(&s_best[s], c);
      const int64_t oi = *cl.map_shared_rank(&s_at[s], c);
      if (c == 0 || better(ov, oi, best, at)) best = ov, at = oi;
    }
    const float first = to_f32(p[0]);
    token = first != first || at == INT64_MAX ? 0 : (int32_t)at;
    if (acc == n || draft[acc] != token) break;
  }
  if (rank == 0) {
    for (int i = tid; i <= a.K; i += kThreads) out[i] = i < acc ? draft[i] : i == acc ? token : -1;
    if (tid == 0) a.accepted[b] = acc;
  }
  cl.sync();  // no CTA leaves while another still reads its best
}

// CTAs a sequence: enough that all SMs read, each with some thousand tokens of its own.
int cluster_size(int64_t seqs, int64_t V) {
  int c = 1;
  while (c < 8 && seqs * c < num_sms() && V > (int64_t)c * 4096) c *= 2;
  return c;
}

template <typename Kernel, typename... Args>
cudaError_t launch_clusters(Kernel kernel, int64_t seqs, int cluster, size_t smem, cudaStream_t st,
                            Args... args) {
  if (smem > 48 * 1024) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(seqs * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  kernel_launch_count()++;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
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
  const size_t smem = (size_t)nb * sizeof(double);
  if (smem > 200 * 1024)
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "vtq_verify_draft: not implemented (vocab too large)");
  cudaError_t e = a->dtype == VTQ_F32 ? launch_clusters(verify_draft_kernel<float>, a->seqs, c, smem, st, p, nb)
                  : a->dtype == VTQ_F16
                      ? launch_clusters(verify_draft_kernel<__half>, a->seqs, c, smem, st, p, nb)
                      : launch_clusters(verify_draft_kernel<__nv_bfloat16>, a->seqs, c, smem, st, p, nb);
  return serve_cuda(e, "vtq_verify_draft");
}

vtq_status vtq_verify_greedy(const vtq_verify_args* a, void* stream) {
  if (vtq_status s = check("vtq_verify_greedy", a, true)) return s;
  if (a->seqs == 0) return VTQ_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int c = cluster_size(a->seqs, a->vocab);
  const VerifyParams p = params(a);
  cudaError_t e = a->dtype == VTQ_F32 ? launch_clusters(verify_greedy_kernel<float>, a->seqs, c, 0, st, p)
                  : a->dtype == VTQ_F16 ? launch_clusters(verify_greedy_kernel<__half>, a->seqs, c, 0, st, p)
                                        : launch_clusters(verify_greedy_kernel<__nv_bfloat16>, a->seqs, c, 0, st, p);
  return serve_cuda(e, "vtq_verify_greedy");
}

}  // extern "C"
