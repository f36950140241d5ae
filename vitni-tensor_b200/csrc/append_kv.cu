// append_kv.cu -- new keys and values into a paged cache, rotated by position on the way, and the
// queries of the same tokens rotated beside them.
//
//   (a, b) -> (a cos - b sin, a sin + b cos),  cos / sin of pos * frequency from a 32-bit table
//
// Bound: HBM by bytes (each input read once, each output written once), latency for a decode step; as it is, issue slots
// (65 % filled, 100 instructions a unit of four f32 values, cos and sin loaded for every head) come before HBM. A
// thread takes a unit: 16 bytes of neighbouring values (and, where the pairs are (i, i + rot / 2), the 16
// bytes of their partners), so that a warp's loads and stores are whole lines: two neighbouring 16-byte
// pieces a thread instead keep L1 half busy with the same sectors twice.
#include <algorithm>

#include "serve.h"
#include "tc5.cuh"

namespace vtq {
namespace {

struct AppendParams {
  vtq_append_kv_args a;
  int rot_units, rest_units;  // of one q / k head: rotated units, units of W other values
  int v_units;                // of one v head
  int units;                  // of a token
};

// W consecutive values as they lie in memory; WIDE: in 16-byte pieces.
template <typename X, int W, bool WIDE>
struct alignas(WIDE ? 16 : sizeof(X)) Raw {
  X v[W];
};
template <typename X, int W, bool WIDE>
__device__ __forceinline__ Raw<X, W, WIDE> load_raw(const X* p) {
  Raw<X, W, WIDE> r;
  if constexpr (WIDE) {
    static_assert(sizeof(X) * W == 16, "one load");
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < W; i++) r.v[i] = p[i];
  }
  return r;
}

template <typename C, int W, bool WIDE>
__device__ __forceinline__ void store(C* p, const float (&v)[W]) {
  if constexpr (WIDE) {
    struct alignas(2 * W) {
      C e[W];
    } w;
#pragma unroll
    for (int i = 0; i < W; i++) w.e[i] = from_f32<C>(v[i]);
    if constexpr (W == 8) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(&w);
    else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(&w);
  } else {
#pragma unroll
    for (int i = 0; i < W; i++) p[i] = from_f32<C>(v[i]);
  }
}

// P pairs' (cos, sin).
template <int P, bool WIDE>
__device__ __forceinline__ void load_turn(const float* cs, float (&c)[P], float (&s)[P]) {
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < P; i += 2) {
      const float4 w = *reinterpret_cast<const float4*>(cs + 2 * i);
      c[i] = w.x, s[i] = w.y, c[i + 1] = w.z, s[i + 1] = w.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < P; i++) {
      const float2 w = *reinterpret_cast<const float2*>(cs + 2 * i);
      c[i] = w.x;
      s[i] = w.y;
    }
  }
}

// Where a token goes: offsets of its slot in the caches (-1: nowhere) and its position (-1: the token is
// left out altogether).
struct Place {
  int64_t k, v;
  int pos;
};
__device__ __forceinline__ Place place_of(const vtq_append_kv_args& a, int64_t t) {
  Place w{-1, -1, -1};
  const int seq = a.seq[t];
  if (seq < 0) return w;  // padding
  const int pos = a.pos[t], page_size = (int)a.kv.page_size;
  int64_t page = -1;
  if (pos >= 0 && (!a.rope || pos < a.max_pos)) {
    w.pos = pos;
    if (seq < a.kv.seqs && pos / page_size < a.kv.table_width) page = a.kv.table[seq * a.kv.table_ld + pos / page_size];
  }
  if (page >= 0 && page < a.kv.pages) {
    w.k = page * a.kv.k_page + pos % page_size * a.kv.k_slot;
    w.v = page * a.kv.v_page + pos % page_size * a.kv.v_slot;
  } else if (a.status) {
    atomicOr(a.status, SERVE_BAD_INDEX);
  }
  return w;
}

// A CTA takes an even share of the tokens, TOK at a time: one thread a token finds its place, then every
// thread has its unit of U tokens at a time, the next ones' values on their way. 28 us on 8081 tokens of
// 32 + 2 x 4 fp32 heads of 64 (4.4 TB/s); 51 us where every thread finds the place itself, by its divisions.
// HALF: a unit is W values and their W partners; otherwise W values, pairs of neighbours.
template <typename X, typename C, int W, int TOK, bool HALF, bool WIDE>
__global__ void __launch_bounds__(TOK > 1 ? 256 : 512, TOK > 1 ? 4 : 1) append_kernel(const __grid_constant__ AppendParams p) {
  tc5::grid_wait();
  constexpr int P = HALF ? W : W / 2;  // pairs of a rotated unit
  constexpr int U = TOK < 4 ? TOK : HALF ? (W == 8 ? 1 : 2) : W == 8 ? 2 : 4;
  __shared__ Place s_place[TOK];
  const vtq_append_kv_args& a = p.a;
  const int head_units = p.rot_units + p.rest_units;
  const int q_units = a.q ? (int)a.heads * head_units : 0, k_units = (int)a.kv.kv_heads * head_units;
  const int half = (int)a.rot_dim / 2;
  const int64_t end = TOK == 1 ? blockIdx.x + 1 : a.tokens * (blockIdx.x + 1) / gridDim.x;
  for (int64_t t0 = TOK == 1 ? blockIdx.x : a.tokens * blockIdx.x / gridDim.x; t0 < end; t0 += TOK) {
    const int tokens = TOK == 1 ? 1 : (int)min((int64_t)TOK, end - t0);
    for (int u0 = 0; u0 < p.units; u0 += blockDim.x) {
      const int u = min(u0 + (int)threadIdx.x, p.units - 1);
      const X* src;
      C* out;
      int64_t src_tok;
      int at, h;  // unit within the head, head
      int kind;   // 0 q, 1 k, 2 v
      if (u < q_units) {
        kind = 0, h = u / head_units, at = u - h * head_units;
        src = static_cast<const X*>(a.q) + h * a.q_head, src_tok = a.q_tok;
        out = static_cast<C*>(a.q_out) + t0 * a.qo_tok + h * a.qo_head;
      } else if (u < q_units + k_units) {
        kind = 1, h = (u - q_units) / head_units, at = u - q_units - h * head_units;
        src = static_cast<const X*>(a.k) + h * a.k_head, src_tok = a.k_tok;
        out = static_cast<C*>(a.kv.k) + h * a.kv.k_head;
      } else {
        kind = 2, h = (u - q_units - k_units) / p.v_units, at = u - q_units - k_units - h * p.v_units;
        src = static_cast<const X*>(a.v) + h * a.v_head, src_tok = a.v_tok;
        out = static_cast<C*>(a.kv.v) + h * a.kv.v_head;
      }
      const bool mine = u0 + (int)threadIdx.x < p.units, turn = kind < 2 && at < p.rot_units;
      const int e = turn || kind == 2 ? at * W : (int)a.rot_dim + (at - p.rot_units) * W;
      src += t0 * src_tok + e;
      out += e;
      const float* cs = a.rope + at * P * 2;
      Raw<X, W, WIDE> x[U], y[HALF ? U : 1];
      auto load = [&](int i0) {
#pragma unroll
        for (int i = 0; i < U; i++) {
          const int t = min(i0 + i, tokens - 1);
          x[i] = load_raw<X, W, WIDE>(src + t * src_tok);
          if (HALF && turn) y[HALF ? i : 0] = load_raw<X, W, WIDE>(src + t * src_tok + half);
        }
      };
      load(0);
      Place only{};  // one token: every thread finds its place itself, rather than wait for one that does
      if constexpr (TOK == 1) {
        only = place_of(a, t0);
      } else if (u0 == 0) {
        __syncthreads();  // the places before have been used
        if (threadIdx.x < tokens) s_place[threadIdx.x] = place_of(a, t0 + threadIdx.x);
        __syncthreads();
      }
      for (int i0 = 0; i0 < tokens; i0 += U) {
        Raw<X, W, WIDE> x0[U], y0[HALF ? U : 1];
        float c[U][P], s[U][P];
#pragma unroll
        for (int i = 0; i < U; i++) {
          x0[i] = x[i];
          if (HALF) y0[HALF ? i : 0] = y[HALF ? i : 0];
          const int pos = TOK == 1 ? only.pos : s_place[min(i0 + i, tokens - 1)].pos;
          if (turn) load_turn<P, WIDE>(cs + (int64_t)max(pos, 0) * half * 2, c[i], s[i]);
        }
        if (i0 + U < tokens) load(i0 + U);
#pragma unroll
        for (int i = 0; i < U; i++) {
          if (!mine || i0 + i >= tokens) continue;
          const Place& w = TOK == 1 ? only : s_place[i0 + i];
          const int64_t to = kind == 0 ? (w.pos < 0 ? -1 : (i0 + i) * a.qo_tok) : kind == 1 ? w.k : w.v;
          if (to < 0) continue;
          float r[W];
#pragma unroll
          for (int k = 0; k < W; k++) r[k] = to_f32(x0[i].v[k]);
          if (turn) {
            if constexpr (HALF) {
              float o[W];
#pragma unroll
              for (int k = 0; k < W; k++) {
                const float b = to_f32(y0[i].v[k]);
                o[k] = r[k] * s[i][k] + b * c[i][k];
                r[k] = r[k] * c[i][k] - b * s[i][k];
              }
              store<C, W, WIDE>(out + to + half, o);
            } else {
#pragma unroll
              for (int k = 0; k < P; k++) {
                const float b = r[2 * k + 1];
                r[2 * k + 1] = r[2 * k] * s[i][k] + b * c[i][k];
                r[2 * k] = r[2 * k] * c[i][k] - b * s[i][k];
              }
            }
          }
          store<C, W, WIDE>(out + to, r);
        }
      }
    }
  }
}

template <typename X, typename C, int W, bool HALF, bool WIDE>
cudaError_t run(const vtq_append_kv_args& a, cudaStream_t st) {
  const int dim = (int)a.kv.head_dim, rot = (int)a.rot_dim;
  AppendParams p;
  p.a = a;
  p.rot_units = rot / (HALF ? 2 * W : W);
  p.rest_units = (dim - rot) / W;
  p.v_units = dim / W;
  p.units = (int)((a.q ? a.heads : 0) + a.kv.kv_heads) * (p.rot_units + p.rest_units) + (int)a.kv.kv_heads * p.v_units;
  // Even passes over a token's units: of 512 threads for one token (latency), of 256 where several CTAs have
  // to fit an SM.
  const bool many = a.tokens > 4 * num_sms();
  const int most = many ? 256 : 512, passes = (p.units + most - 1) / most;
  const int threads = ((p.units + passes - 1) / passes + 31) / 32 * 32;
  // A decode step's few tokens go one to a CTA, for latency; many in even shares to as many as fit at once.
  if (many)
    return launch_after(append_kernel<X, C, W, 32, HALF, WIDE>, dim3((unsigned)(num_sms() * std::max(1, 1024 / threads))),
                        threads, 0, 1, st, p);
  return launch_after(append_kernel<X, C, W, 1, HALF, WIDE>, dim3((unsigned)a.tokens), threads, 0, 1, st, p);
}

template <typename X, typename C>
cudaError_t launch(const vtq_append_kv_args& a, cudaStream_t st) {
  constexpr int W = 16 / sizeof(X);
  const bool by_half = a.flags & VTQ_ROPE_HALF;
  const int dim = (int)a.kv.head_dim, rot = (int)a.rot_dim;
  // 16-byte loads where every head begins on one and units come whole.
  auto fits = [](const void* p, int64_t s0, int64_t s1, int64_t m) { return aligned16(p) && s0 % m == 0 && s1 % m == 0; };
  const bool wide = rot % (by_half ? 2 * W : W) == 0 && (dim - rot) % W == 0 && aligned16(a.rope) &&
                    fits(a.k, a.k_tok, a.k_head, W) && fits(a.v, a.v_tok, a.v_head, W) &&
                    (!a.q || (fits(a.q, a.q_tok, a.q_head, W) && fits(a.q_out, a.qo_tok, a.qo_head, W)));
  if (by_half) return wide ? run<X, C, W, true, true>(a, st) : run<X, C, 1, true, false>(a, st);
  return wide ? run<X, C, W, false, true>(a, st) : run<X, C, 2, false, false>(a, st);
}

}  // namespace

vtq_status serve_check_kv(const char* fn, const vtq_paged_kv& kv) {
  if (kv.dtype != VTQ_F16 && kv.dtype != VTQ_BF16)
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (cache not F16 / BF16)", fn);
  if (kv.pages < 0 || kv.page_size < 1 || kv.kv_heads < 1 || kv.head_dim < 1 || kv.seqs < 0 ||
      kv.table_width < 0 || kv.pages > INT32_MAX || kv.page_size > INT32_MAX)
    return serve_fail(VTQ_ERR_INTERNAL, "%s: bad cache shape", fn);
  if (kv.head_dim % 8 || kv.head_dim > 256 || kv.kv_heads > 4096)
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED,
                      "%s: not implemented (head_dim not a multiple of 8 up to 256, or over 4096 heads)", fn);
  // (The table is read before a page's number is compared with how many there are.)
  if ((kv.pages && (!kv.k || !kv.v)) || (!kv.table && kv.seqs && kv.table_width))
    return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null cache pointer", fn);
  if (!aligned16(kv.k) || !aligned16(kv.v) || kv.k_page % 8 || kv.k_slot % 8 || kv.k_head % 8 ||
      kv.v_page % 8 || kv.v_slot % 8 || kv.v_head % 8)
    return serve_fail(VTQ_ERR_INTERNAL, "%s: cache not 16-byte aligned, or strides not multiples of 8", fn);
  return VTQ_OK;
}

}  // namespace vtq

using namespace vtq;

extern "C" vtq_status vtq_append_kv(const vtq_append_kv_args* a, void* stream) {
  const char* fn = "vtq_append_kv";
  if (!a) return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null arguments", fn);
  if (vtq_status s = serve_check_kv(fn, a->kv)) return s;
  if (!serve_elt(a->x_dtype))
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (k / v not F32 / F16 / BF16)", fn);
  if (a->tokens < 0 || a->tokens > INT32_MAX || (a->q && (a->heads < 1 || a->heads > 65536)))
    return serve_fail(VTQ_ERR_INTERNAL, "%s: bad shape", fn);
  if (a->rot_dim < 0 || a->rot_dim % 2 || a->rot_dim > a->kv.head_dim || (a->rope ? a->rot_dim < 2 : a->rot_dim != 0))
    return serve_fail(VTQ_ERR_INTERNAL, "%s: rot_dim not an even number up to head_dim (0 without rope)", fn);
  if (a->rope && (a->max_pos < 1 || (reinterpret_cast<uintptr_t>(a->rope) & 7u)))
    return serve_fail(VTQ_ERR_INTERNAL, "%s: bad rope table", fn);
  if (a->tokens == 0) return VTQ_OK;
  if (!a->k || !a->v || !a->seq || !a->pos || (a->q && !a->q_out))
    return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null pointer", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = a->kv.dtype == VTQ_BF16;
  cudaError_t e = a->x_dtype == VTQ_F32   ? (bf ? launch<float, __nv_bfloat16>(*a, st) : launch<float, __half>(*a, st))
                  : a->x_dtype == VTQ_F16 ? (bf ? launch<__half, __nv_bfloat16>(*a, st) : launch<__half, __half>(*a, st))
                                          : (bf ? launch<__nv_bfloat16, __nv_bfloat16>(*a, st)
                                                : launch<__nv_bfloat16, __half>(*a, st));
  return serve_cuda(e, fn);
}
