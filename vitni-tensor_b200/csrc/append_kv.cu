// append_kv.cu -- new keys and values into a paged cache, rotated by position on the way, and the
// queries of the same tokens rotated beside them.
//
//   (a, b) -> (a cos - b sin, a sin + b cos),  cos / sin of pos * frequency from a 32-bit table
//
// Bound: HBM by bytes (each input read once, each output written once), latency for a decode step.
// One CTA takes one token; each of its threads takes one unit of 16 values (a rotated unit: 8 pairs)
// or 8 (values that are not rotated), so that a decode step has every load in flight at once: the
// inputs' loads do not wait for the table's, which need pos, seq and the page number first.
#include <algorithm>

#include "serve.h"
#include "vtq_internal.h"

namespace vtq {
namespace {

struct AppendParams {
  vtq_append_kv_args a;
  int rot_units, rest_units;  // of one q / k head: units of 2 VEC rotated values, units of VEC others
  int v_units;                // of one v head: units of VEC values
  int units;                  // of a token
};

// VEC consecutive values as 32-bit floats.
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
  if constexpr (VEC == 8 && sizeof(T) == 2) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = to_f32(e[i]);
  } else if constexpr (VEC == 8) {
    const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i++) v[i] = to_f32(p[i]);
  }
}

template <typename C, int VEC>
__device__ __forceinline__ void store_vec(C* p, const float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    uint4 w;
    C* e = reinterpret_cast<C*>(&w);
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = from_f32<C>(v[i]);
    *reinterpret_cast<uint4*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i++) p[i] = from_f32<C>(v[i]);
  }
}

template <typename X, typename C, int VEC>
__global__ void __launch_bounds__(512) append_kernel(const __grid_constant__ AppendParams p) {
  const vtq_append_kv_args& a = p.a;
  const int64_t t = blockIdx.x;
  const int seq = a.seq[t], pos = a.pos[t];
  if (seq < 0) return;  // padding
  const int head_units = p.rot_units + p.rest_units;
  const int q_units = a.q ? (int)a.heads * head_units : 0, k_units = (int)a.kv.kv_heads * head_units;
  const int half = (int)a.rot_dim / 2;
  const bool by_half = a.flags & VTQ_ROPE_HALF;
  bool turnable = pos >= 0 && (!a.rope || pos < a.max_pos);
  int64_t page = -1;
  if (turnable && seq < a.kv.seqs && pos / a.kv.page_size < a.kv.table_width) {
    page = a.kv.table[seq * a.kv.table_ld + pos / a.kv.page_size];
    if (page >= a.kv.pages) page = -1;
  }
  const int64_t slot = pos >= 0 ? pos % a.kv.page_size : 0;
  if (page < 0 && threadIdx.x == 0 && a.status) atomicOr(a.status, SERVE_BAD_INDEX);
  if (!turnable) return;
  for (int u = threadIdx.x; u < p.units; u += blockDim.x) {
    const X* src;
    C* dst = nullptr;
    int at;  // unit within the head
    bool is_v = false;
    if (u < q_units) {
      const int h = u / head_units;
      at = u - h * head_units;
      src = static_cast<const X*>(a.q) + t * a.q_tok + h * a.q_head;
      dst = static_cast<C*>(a.q_out) + t * a.qo_tok + h * a.qo_head;
    } else if (u < q_units + k_units) {
      const int h = (u - q_units) / head_units;
      at = u - q_units - h * head_units;
      src = static_cast<const X*>(a.k) + t * a.k_tok + h * a.k_head;
      if (page >= 0) dst = static_cast<C*>(a.kv.k) + page * a.kv.k_page + slot * a.kv.k_slot + h * a.kv.k_head;
    } else {
      const int h = (u - q_units - k_units) / p.v_units;
      at = u - q_units - k_units - h * p.v_units;
      src = static_cast<const X*>(a.v) + t * a.v_tok + h * a.v_head;
      if (page >= 0) dst = static_cast<C*>(a.kv.v) + page * a.kv.v_page + slot * a.kv.v_slot + h * a.kv.v_head;
      is_v = true;
    }
    if (!is_v && at < p.rot_units) {
      // VEC pairs: (i, i + half), or two neighbours.
      const int e0 = by_half ? at * VEC : 2 * at * VEC, e1 = by_half ? e0 + half : e0 + VEC;
      float x[VEC], y[VEC], c[VEC], s[VEC];
      load_vec<X, VEC>(src + e0, x);
      load_vec<X, VEC>(src + e1, y);
      const float* cs = a.rope + ((int64_t)pos * half + at * VEC) * 2;
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        const float2 w = *reinterpret_cast<const float2*>(cs + 2 * i);
        c[i] = w.x;
        s[i] = w.y;
      }
      float r0[VEC], r1[VEC];
      if (by_half) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          r0[i] = x[i] * c[i] - y[i] * s[i];
          r1[i] = x[i] * s[i] + y[i] * c[i];
        }
      } else {
        float z[2 * VEC], r[2 * VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) z[i] = x[i], z[VEC + i] = y[i];
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          r[2 * i] = z[2 * i] * c[i] - z[2 * i + 1] * s[i];
          r[2 * i + 1] = z[2 * i] * s[i] + z[2 * i + 1] * c[i];
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) r0[i] = r[i], r1[i] = r[VEC + i];
      }
      if (dst) {
        store_vec<C, VEC>(dst + e0, r0);
        store_vec<C, VEC>(dst + e1, r1);
      }
    } else {
      const int e0 = is_v ? at * VEC : (int)a.rot_dim + (at - p.rot_units) * VEC;
      float x[VEC];
      load_vec<X, VEC>(src + e0, x);
      if (dst) store_vec<C, VEC>(dst + e0, x);
    }
  }
}

template <typename X, typename C>
cudaError_t launch(const vtq_append_kv_args& a, cudaStream_t st) {
  const int dim = (int)a.kv.head_dim, rot = (int)a.rot_dim;
  // 16-byte accesses where every head begins on one and the pairs come in whole units.
  constexpr int kX = 16 / sizeof(X);
  auto strides_ok = [](int64_t s0, int64_t s1, int64_t m) { return s0 % m == 0 && s1 % m == 0; };
  const bool wide = ((a.flags & VTQ_ROPE_HALF) ? rot % 16 == 0 : rot % 16 == 0) && (dim - rot) % 8 == 0 &&
                    aligned16(a.k) && aligned16(a.v) && strides_ok(a.k_tok, a.k_head, kX) &&
                    strides_ok(a.v_tok, a.v_head, kX) &&
                    (!a.q || (aligned16(a.q) && aligned16(a.q_out) && strides_ok(a.q_tok, a.q_head, kX) &&
                              strides_ok(a.qo_tok, a.qo_head, 8)));
  const int vec = wide ? 8 : 1;
  AppendParams p;
  p.a = a;
  p.rot_units = rot / (2 * vec);
  p.rest_units = (dim - rot) / vec;
  p.v_units = dim / vec;
  p.units = (int)((a.q ? a.heads : 0) + a.kv.kv_heads) * (p.rot_units + p.rest_units) +
            (int)a.kv.kv_heads * p.v_units;
  const int threads = std::min(512, (p.units + 31) / 32 * 32);
  kernel_launch_count()++;
  if (wide) append_kernel<X, C, 8><<<(unsigned)a.tokens, threads, 0, st>>>(p);
  else append_kernel<X, C, 1><<<(unsigned)a.tokens, threads, 0, st>>>(p);
  return cudaGetLastError();
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
  if (kv.pages && (!kv.k || !kv.v || (!kv.table && kv.seqs * kv.table_width)))
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
  if (a->rope && (a->max_pos < 0 || (reinterpret_cast<uintptr_t>(a->rope) & 7u)))
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
