// linear_i8.cu -- 8-bit linears over a batch of tokens: codes and a scale for each token, signed
// 8-bit weights with a scale for each output channel.
//
//   y[t][o] = (sum_i q[t][i] w[o][i]) * (x_scale[t] w_scale[o]) + bias[o]
//
// The sum is a contraction of signed bytes on the tensor cores (tcgen05.mma kind::i8, 32-bit
// accumulators in TMEM): exact, so the split over K and the order of the parts do not show.
//
// The weights are the MMA's rows (M = 128 output channels) and the tokens its columns (N = 16 .. 256):
// a few tokens then waste columns that cost nothing to load, and a lane of TMEM is one output channel,
// so that a warp's store of one column is 32 neighbouring channels of one token.
#include <cooperative_groups.h>

#include <algorithm>

#include "serve.h"
#include "tc5.cuh"
#include "vtq_internal.h"

namespace cg = cooperative_groups;

namespace vtq {
namespace {

// ---- codes and scales of the tokens ----

constexpr int kQThreads = 512, kQKeep = 4;  // values kept in registers: 4 x 8 a thread

// Round-half-even of the real quotient x / s, as the low byte of a word. x / s is first rounded as the
// product with 1 / s, by adding 1.5 * 2^23, whose last bits are then the whole number: at most one off. The
// remainder x - q s is exact in 32 bits (both are multiples of a common power of two and it is no larger
// than s), so comparing it with s / 2 tells whether q was right; only quotients next to a half get there.
__device__ __forceinline__ uint32_t code(float x, float s, float inv, float look) {
  constexpr float kMagic = 12582912.0f;
  float t = fmaf(x, inv, kMagic);
  const float q = __fsub_rn(t, kMagic), rem = fmaf(-q, s, x);
  if (fabsf(rem) >= look) {
    const float h = 0.5f * s;
    const bool odd = ((int)q) & 1;
    if (rem > h || (rem == h && odd)) t = __fadd_rn(t, 1.0f);
    else if (rem < -h || (rem == -h && odd)) t = __fsub_rn(t, 1.0f);
    // A scale rounded down in the subnormals leaves quotients over 127.
    t = fminf(fmaxf(t, kMagic - 127.0f), kMagic + 127.0f);
  }
  return __float_as_uint(t);
}

template <typename X>
__device__ __forceinline__ void load8(const X* row, int64_t i, int64_t n, bool wide, float (&v)[8]) {
  if (wide && i + 8 <= n) {
    if constexpr (sizeof(X) == 2) {
      const uint4 w = *reinterpret_cast<const uint4*>(row + i);
      const X* e = reinterpret_cast<const X*>(&w);
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = to_f32(e[k]);
    } else {
      const float4 a = *reinterpret_cast<const float4*>(row + i), b = *reinterpret_cast<const float4*>(row + i + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = i + k < n ? to_f32(row[i + k]) : 0.0f;
  }
}

// One CTA a token. Values of up to 16384 inputs stay in registers between the two passes.
template <typename X>
__global__ void __launch_bounds__(kQThreads)
    quantize_kernel(const X* __restrict__ x, int64_t ldx, int64_t n, bool wide, int8_t* __restrict__ q,
                    int64_t ldq, bool wide_q, float* __restrict__ scale) {
  __shared__ uint32_t s_max[kQThreads / 32];
  tc5::grid_wait();
  tc5::grid_release();
  const X* row = x + (int64_t)blockIdx.x * ldx;
  int8_t* out = q + (int64_t)blockIdx.x * ldq;
  const int64_t step = (int64_t)blockDim.x * 8, i0 = (int64_t)threadIdx.x * 8;
  float keep[kQKeep][8];
  uint32_t m = 0;  // |x| as bits: ordered as the values, infinities and NaN above all
#pragma unroll
  for (int k = 0; k < kQKeep; k++) {
    if (i0 + k * step < n) {
      load8(row, i0 + k * step, n, wide, keep[k]);
#pragma unroll
      for (int e = 0; e < 8; e++) m = max(m, __float_as_uint(keep[k][e]) & 0x7fffffffu);
    }
  }
  for (int64_t i = i0 + kQKeep * step; i < n; i += step) {
    float v[8];
    load8(row, i, n, wide, v);
#pragma unroll
    for (int e = 0; e < 8; e++) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
  m = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); w++) m = max(m, s_max[w]);
  const bool finite = m < 0x7f800000u;
  float s = finite ? __fdiv_rn(__uint_as_float(m), 127.0f) : __uint_as_float(0x7fc00000u);
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
  const bool some = finite && s > 0.0f;
  const bool tiny = s < 1e-30f;
  const float up = tiny ? 18446744073709551616.0f : 1.0f;  // keeps 1 / s finite; exact on both
  s = s * up;
  const float look = tiny ? 0.0f : 0.5f * s;  // 0: every quotient is looked at, for those over 127
  const float inv = some ? __fdiv_rn(1.0f, s) : 0.0f;
  auto put = [&](int64_t i, const float (&v)[8]) {
    uint32_t c[8], w[2] = {0, 0};
    if (some) {
#pragma unroll
      for (int e = 0; e < 8; e++) c[e] = code(tiny ? v[e] * up : v[e], s, inv, look);
#pragma unroll
      for (int e = 0; e < 2; e++)
        w[e] = __byte_perm(__byte_perm(c[4 * e], c[4 * e + 1], 0x0040), __byte_perm(c[4 * e + 2], c[4 * e + 3], 0x0040), 0x5410);
    }
    if (wide_q && i + 8 <= n) {
      *reinterpret_cast<uint2*>(out + i) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (i + e < n) out[i + e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
    }
  };
#pragma unroll
  for (int k = 0; k < kQKeep; k++)
    if (i0 + k * step < n) put(i0 + k * step, keep[k]);
  for (int64_t i = i0 + kQKeep * step; i < n; i += step) {
    float v[8];
    load8(row, i, n, wide, v);
    put(i, v);
  }
}

template <typename X>
cudaError_t launch_quantize(const X* x, int64_t ldx, int64_t tokens, int64_t n, int8_t* q, int64_t ldq,
                            float* scale, cudaStream_t st) {
  const bool wide = aligned16(x) && ldx % (16 / (int)sizeof(X)) == 0;
  const bool wide_q = (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ldq % 8 == 0;
  // Few tokens: a row over as many threads as it has 16 bytes for, for latency. Many: 32 values a thread, so
  // that more rows are in flight.
  const int64_t each = tokens <= 2 * num_sms() ? 8 : 32;
  const int threads = (int)std::min<int64_t>(kQThreads, std::max<int64_t>(32, ((n + each - 1) / each + 31) / 32 * 32));
  return launch_after(quantize_kernel<X>, dim3((unsigned)tokens), threads, 0, 1, st, x, ldx, n, wide, q, ldq, wide_q, scale);
}

cudaError_t quantize(int dtype, const void* x, int64_t ldx, int64_t tokens, int64_t n, int8_t* q, int64_t ldq,
                     float* scale, cudaStream_t st) {
  if (dtype == VTQ_F32) return launch_quantize(static_cast<const float*>(x), ldx, tokens, n, q, ldq, scale, st);
  if (dtype == VTQ_F16) return launch_quantize(static_cast<const __half*>(x), ldx, tokens, n, q, ldq, scale, st);
  return launch_quantize(static_cast<const __nv_bfloat16*>(x), ldx, tokens, n, q, ldq, scale, st);
}

// ---- the product ----

struct I8Params {
  int T, K, N;
  int kblocks;  // of 128 inputs
  bool early;   // the kernel before is this call's own: whatever wrote the weights has ended
  const float* xs;
  const float* ws;
  const float* bias;
  void* y;
  int64_t ldy;
  unsigned* status;
};

constexpr int BM = 128;          // output channels a tile
constexpr uint32_t A_STAGE = BM * 128;
constexpr int kThreads = 192;    // producer warp, MMA warp, 4 epilogue warps

__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one));
}

// A sum as a float. Only 131072 products of -128 and -128 leave the range of 32 bits: their sum, 2^31, is held as the
// lowest value, one that no other sum has (the lowest of those is 131072 x 127 x -128).
constexpr int kMostInputs = 131072;
__device__ __forceinline__ float sum_f32(int acc) { return acc == INT32_MIN ? 2147483648.0f : __int2float_rn(acc); }

template <typename Y>
__device__ __forceinline__ void store_y(const I8Params& p, int t, int o, int acc, float wsc, float b) {
  float v = sum_f32(acc) * (p.xs[t] * wsc);
  if (p.bias) v += b;
  static_cast<Y*>(p.y)[(int64_t)t * p.ldy + o] = from_f32<Y>(v);
}

// One tile of 128 channels x NT tokens; the CTAs of a cluster share its K and add their integer parts
// through each other's shared memory.
template <int NT, int STAGES, typename Y>
__global__ void __launch_bounds__(kThreads)
    i8_tile_kernel(const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmx,
                   const __grid_constant__ I8Params p) {
  constexpr uint32_t B_STAGE = NT * 128, STAGE = A_STAGE + B_STAGE;
  constexpr uint32_t COLS = NT < 32 ? 32 : NT;
  constexpr uint32_t kIdesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
  static_assert(STAGES * STAGE >= BM * NT * 4, "the parts reuse the stages");
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_bar[2 * STAGES + 1];
  __shared__ uint32_t s_slot;
  __shared__ int s_abort;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  int* part = reinterpret_cast<int*>(smem_raw + (base - smem_u32(smem_raw)));
  auto FULL = [&](int i) { return smem_u32(&s_bar[i]); };
  auto EMPTY = [&](int i) { return smem_u32(&s_bar[STAGES + i]); };
  const uint32_t DONE = smem_u32(&s_bar[2 * STAGES]);
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), splits = (int)cl.num_blocks();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int o0 = (int)(blockIdx.x / splits) * BM, t0 = (int)blockIdx.y * NT;
  const int kb0 = (int)((int64_t)p.kblocks * rank / splits), kb1 = (int)((int64_t)p.kblocks * (rank + 1) / splits);
  const int nk = kb1 - kb0;
  volatile int* abort_flag = &s_abort;

  if (tid == 0) {
    for (int i = 0; i < STAGES; i++) {
      tc5::bar_init(FULL(i), 1);
      tc5::bar_init(EMPTY(i), 1);
    }
    tc5::bar_init(DONE, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tc5::alloc(smem_u32(&s_slot), COLS);
  tc5::fence_before();
  __syncthreads();
  tc5::fence_after();
  const uint32_t tmem = s_slot;
  auto fail = [&]() {
    record_error(p.status, KERR_TIMEOUT);
    *abort_flag = 1;
  };

  if (warp == 0) {
    if (lane == 0) {
      // The call's own codes kernel lets this one begin only when all before it have ended: as many weights
      // as fit are on their way before its codes are waited for. With the caller's codes the kernel
      // before may be the one that writes the weights.
      if (!p.early) tc5::grid_wait();
      const int ahead = min(nk, STAGES);
      for (int k = 0; k < ahead; k++) {
        tc5::bar_expect(FULL(k), STAGE);
        tc5::tma_2d(base + k * STAGE, &tmw, (kb0 + k) * 128, o0, FULL(k));
      }
      tc5::grid_wait();
      for (int k = 0; k < ahead; k++)
        tc5::tma_2d(base + k * STAGE + A_STAGE, &tmx, (kb0 + k) * 128, t0, FULL(k));
      for (int k = ahead; k < nk; k++) {
        const int s = k % STAGES;
        if (!tc5::bar_wait(EMPTY(s), ((k / STAGES) + 1) & 1)) {
          fail();
          break;
        }
        tc5::bar_expect(FULL(s), STAGE);
        tc5::tma_2d(base + s * STAGE, &tmw, (kb0 + k) * 128, o0, FULL(s));
        tc5::tma_2d(base + s * STAGE + A_STAGE, &tmx, (kb0 + k) * 128, t0, FULL(s));
      }
    }
  } else if (warp == 1) {
    const uint32_t one = tc5::elect();
    for (int k = 0; k < nk; k++) {
      const int s = k % STAGES;
      if (!tc5::bar_wait(FULL(s), (k / STAGES) & 1)) {
        if (lane == 0) fail();
        break;
      }
      tc5::fence_after();
      const uint32_t sa = base + s * STAGE, sb = sa + A_STAGE;
#pragma unroll
      for (int c = 0; c < 4; c++)
        mma_i8(tmem, tc5::desc_sw128(sa + 32 * c), tc5::desc_sw128(sb + 32 * c), kIdesc, (k | c) ? 1u : 0u, one);
      tc5::commit(EMPTY(s), one);
    }
    tc5::commit(DONE, one);
  } else {
    tc5::grid_wait();  // the token scales
    const bool ok = tc5::bar_wait(DONE, 0);
    if (!ok && lane == 0) fail();
    tc5::fence_after();
    const int quad = warp & 3, row = 32 * quad + lane, o = o0 + row;
    const float wsc = o < p.N ? p.ws[o] : 0.0f, b = p.bias && o < p.N ? p.bias[o] : 0.0f;
#pragma unroll 1
    for (int c = 0; c < NT; c += 16) {
      uint32_t r[16];
      tc5::ld16(tmem + ((uint32_t)(32 * quad) << 16) + c, r);
      tc5::wait_ld();
      if (splits == 1) {
        if (ok && !*abort_flag && o < p.N) {
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (t0 + c + i < p.T) store_y<Y>(p, t0 + c + i, o, (int)r[i], wsc, b);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; i++) part[(c + i) * BM + row] = nk ? (int)r[i] : 0;
      }
    }
    tc5::fence_before();
  }
  if (*abort_flag) tc5::settle();
  __syncthreads();
  if (warp == 1) {
    tc5::fence_after();
    tc5::dealloc(tmem, COLS);
  }
  if (splits > 1) {
    cl.sync();
    // Token c of the tile is added up by CTA c mod splits: a warp a token, a lane four channels, two tokens'
    // parts from all CTAs in flight at once (one 4-byte load after the other: 60 us at 256 tokens).
    const int o = o0 + 4 * lane;
    float wsc[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      wsc[i] = o + i < p.N ? p.ws[o + i] : 0.0f;
      b[i] = p.bias && o + i < p.N ? p.bias[o + i] : 0.0f;
    }
    const int last = min(NT, p.T - t0);
    for (int c0 = rank + splits * warp; c0 < last; c0 += 2 * splits * (kThreads / 32)) {
      int4 v[2][8];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int c = c0 + h * splits * (kThreads / 32);
#pragma unroll
        for (int s = 0; s < 8; s++)
          if (s < splits && c < last) v[h][s] = reinterpret_cast<const int4*>(cl.map_shared_rank(part, s) + c * BM)[lane];
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int c = c0 + h * splits * (kThreads / 32);
        if (c >= last || *abort_flag) continue;
        uint32_t acc[4] = {0, 0, 0, 0};  // modulo 2^32, as the tensor cores add
#pragma unroll
        for (int s = 0; s < 8; s++)
          if (s < splits) acc[0] += v[h][s].x, acc[1] += v[h][s].y, acc[2] += v[h][s].z, acc[3] += v[h][s].w;
        const float xs = p.xs[t0 + c];
        Y* y = static_cast<Y*>(p.y) + (int64_t)(t0 + c) * p.ldy + o;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float r = sum_f32((int)acc[i]) * (xs * wsc[i]);
          if (p.bias) r += b[i];
          if (o + i < p.N) y[i] = from_f32<Y>(r);
        }
      }
    }
    cl.sync();  // no CTA leaves while another still reads its part
  }
}

// Many tokens: persistent pairs of CTAs (cta_group::2), each walking tiles of 256 channels x 256 tokens. A
// CTA brings 128 channels and 128 tokens, 32 KB for 2^22 products: at the 62 bytes a cycle that L2 gives an
// SM here this feeds the tensor cores, where a CTA by itself (128 x 256, 48 KB) waits: 101 us against 92 on
// 2048 x 4096 x 14336 in runs of some ms, the codes' kernel of 9 us included (94 as it is now, and 109 in runs
// of 0.15 s, when the power limit has lowered the clock). The leader (rank 0) issues the products for both;
// barriers that only it waits for are its own, signalled from the peer. Two accumulators of 256 columns in TMEM,
// so that one tile is stored while the next one is summed; the operand ring runs on across tiles.
constexpr int PM = 256, PN = 256, kPStages = 6, kPEpiWarps = 8, kPThreads = 64 + 32 * kPEpiWarps;
constexpr uint32_t kPHalf = 128 * 128, kPStage = 2 * kPHalf;

__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one));
}
// Arrives at the barrier of this offset in both CTAs once the products so far are done.
__device__ __forceinline__ void commit_pair(uint32_t bar, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b16 m;\n\tsetp.ne.b32 q, %1, 0;\n\tmov.b16 m, 3;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(bar),
      "r"(one)
      : "memory");
}
// The address of a shared location of this CTA's in the pair's leader.
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
// A load into this CTA that completes on a barrier of the leader's.
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
      "{%2, %3}], [%4];" ::"r"(dst),
      "l"(tm), "r"(x), "r"(y), "r"(leader_bar)
      : "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <typename Y>
__global__ void __launch_bounds__(kPThreads, 1)
    i8_wide_kernel(const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmx,
                   const __grid_constant__ I8Params p, int tiles, int token_tiles) {
  constexpr uint32_t kIdesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(PN >> 3) << 17) | ((uint32_t)(PM >> 4) << 24);
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_bar[2 * kPStages + 4];
  __shared__ uint32_t s_slot;
  __shared__ int s_abort;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  auto FULL = [&](int i) { return smem_u32(&s_bar[i]); };                 // the leader's: both CTAs' operands are there
  auto EMPTY = [&](int i) { return smem_u32(&s_bar[kPStages + i]); };     // each CTA's own
  auto ACC_FULL = [&](int i) { return smem_u32(&s_bar[2 * kPStages + i]); };
  auto ACC_EMPTY = [&](int i) { return smem_u32(&s_bar[2 * kPStages + 2 + i]); };  // the leader's
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), first = (int)blockIdx.x / 2, step = (int)gridDim.x / 2;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nk = p.kblocks;
  volatile int* abort_flag = &s_abort;
  if (tid == 0) {
    for (int i = 0; i < kPStages; i++) {
      tc5::bar_init(FULL(i), 1);
      tc5::bar_init(EMPTY(i), 1);
    }
    for (int i = 0; i < 2; i++) {
      tc5::bar_init(ACC_FULL(i), 1);
      tc5::bar_init(ACC_EMPTY(i), 2 * kPEpiWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc5::fence_before();
  cl.sync();
  tc5::fence_after();
  const uint32_t tmem = s_slot;
  auto fail = [&]() {
    record_error(p.status, KERR_TIMEOUT);
    *abort_flag = 1;
  };

  if (warp == 0) {
    if (lane == 0) {
      tc5::grid_wait();  // the codes
      int g = 0;
      for (int u = first; u < tiles && !*abort_flag; u += step) {
        const int o0 = u / token_tiles * PM + rank * 128, t0 = u % token_tiles * PN + rank * 128;
        for (int k = 0; k < nk; k++, g++) {
          const int s = g % kPStages;
          if (g >= kPStages && !tc5::bar_wait(EMPTY(s), tc5::phase(g, kPStages, true))) {
            fail();
            break;
          }
          const uint32_t full = in_leader(FULL(s)), at = base + s * kPStage;
          if (rank == 0) tc5::bar_expect(FULL(s), 2 * kPStage);
          tma_2d_pair(at, &tmw, k * 128, o0, full);
          tma_2d_pair(at + kPHalf, &tmx, k * 128, t0, full);
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t one = tc5::elect();
      int g = 0, n = 0;
      bool ok = true;
      for (int u = first; u < tiles && ok; u += step, n++) {
        const int acc = n & 1;
        ok = n < 2 || tc5::bar_wait(ACC_EMPTY(acc), tc5::phase(n, 2, true));
        for (int k = 0; k < nk && ok; k++, g++) {
          const int s = g % kPStages;
          ok = tc5::bar_wait(FULL(s), tc5::phase(g, kPStages));
          if (!ok) break;
          tc5::fence_after();
          const uint32_t sa = base + s * kPStage, sb = sa + kPHalf;
#pragma unroll
          for (int c = 0; c < 4; c++)
            mma_i8_pair(tmem + acc * PN, tc5::desc_sw128(sa + 32 * c), tc5::desc_sw128(sb + 32 * c), kIdesc, (k | c) ? 1u : 0u, one);
          commit_pair(EMPTY(s), one);
        }
        if (ok) commit_pair(ACC_FULL(acc), one);
      }
      if (!ok && lane == 0) fail();
    }
  } else {
    tc5::grid_wait();  // the token scales
    const int quad = warp & 3, half = (warp - 2) >> 2, row = 32 * quad + lane;
    int n = 0;
    for (int u = first; u < tiles; u += step, n++) {
      const int acc = n & 1, o = u / token_tiles * PM + rank * 128 + row, t0 = u % token_tiles * PN + half * (PN / 2);
      if (!tc5::bar_wait(ACC_FULL(acc), tc5::phase(n, 2))) {
        if (lane == 0) fail();
        break;
      }
      tc5::fence_after();
      const float wsc = o < p.N ? p.ws[o] : 0.0f, b = p.bias && o < p.N ? p.bias[o] : 0.0f;
      Y* y = static_cast<Y*>(p.y) + (int64_t)t0 * p.ldy + o;
      const uint32_t at = tmem + ((uint32_t)(32 * quad) << 16) + acc * PN + half * (PN / 2);
#pragma unroll 1
      for (int c = 0; c < PN / 2; c += 32) {
        uint32_t r[32];
        float xs[32];
        tc5::ld16(at + c, *reinterpret_cast<uint32_t(*)[16]>(r));
        tc5::ld16(at + c + 16, *reinterpret_cast<uint32_t(*)[16]>(r + 16));
        const bool all = t0 + c + 32 <= p.T;
        // Each lane reads one token's scale; they are passed round below.
        const float mine = t0 + c + lane < p.T ? p.xs[t0 + c + lane] : 0.0f;
#pragma unroll
        for (int i = 0; i < 32; i++) xs[i] = __shfl_sync(0xffffffffu, mine, i);
        tc5::wait_ld();
        if (o < p.N) {
          float sum[32];
#pragma unroll
          for (int i = 0; i < 32; i++) sum[i] = __int2float_rn((int)r[i]);
          if (p.K == kMostInputs) {  // (testing every sum costs 1 % on 2048 x 4096 x 14336)
#pragma unroll
            for (int i = 0; i < 32; i++) sum[i] = sum[i] == -2147483648.0f ? 2147483648.0f : sum[i];  // as sum_f32
          }
#pragma unroll
          for (int i = 0; i < 32; i++) {
            float v = sum[i] * (xs[i] * wsc);
            if (p.bias) v += b;
            if (all || t0 + c + i < p.T) y[(int64_t)(c + i) * p.ldy] = from_f32<Y>(v);
          }
        }
      }
      tc5::fence_before();
      __syncwarp();
      if (lane == 0) arrive_remote(in_leader(ACC_EMPTY(acc)));
    }
  }
  if (*abort_flag) tc5::settle();
  tc5::fence_before();
  cl.sync();  // the leader's products read the peer's operands and write its accumulators
  if (warp == 1) {
    tc5::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

template <typename Y>
cudaError_t launch_wide(const CUtensorMap& tmw, const CUtensorMap& tmx, const I8Params& p, cudaStream_t st) {
  constexpr size_t smem = (size_t)kPStages * kPStage + 1024;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem((const void*)i8_wide_kernel<Y>, smem, allowed);
  if (e != cudaSuccess) return e;
  const int token_tiles = (p.T + PN - 1) / PN, tiles = (p.N + PM - 1) / PM * token_tiles;
  return launch_after(i8_wide_kernel<Y>, dim3((unsigned)(2 * std::min(tiles, num_sms() / 2))), kPThreads, smem, 2, st, tmw, tmx, p,
                      tiles, token_tiles);
}

template <int NT, int STAGES, typename Y>
cudaError_t launch_tile(const CUtensorMap& tmw, const CUtensorMap& tmx, const I8Params& p, int splits, cudaStream_t st) {
  constexpr size_t smem = (size_t)STAGES * (A_STAGE + NT * 128) + 1024;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem((const void*)i8_tile_kernel<NT, STAGES, Y>, smem, allowed);
  if (e != cudaSuccess) return e;
  return launch_after(i8_tile_kernel<NT, STAGES, Y>, dim3((unsigned)((p.N + BM - 1) / BM * splits), (unsigned)((p.T + NT - 1) / NT)),
                      kThreads, smem, splits, st, tmw, tmx, p);
}

template <typename Y>
cudaError_t product(const CUtensorMap& tmw, const CUtensorMap& tmx, const I8Params& p, int nt, int splits, cudaStream_t st) {
  switch (nt) {
    case 16: return launch_tile<16, 5, Y>(tmw, tmx, p, splits, st);
    case 32: return launch_tile<32, 5, Y>(tmw, tmx, p, splits, st);
    case 64: return launch_tile<64, 4, Y>(tmw, tmx, p, splits, st);
    case 128: return launch_tile<128, 3, Y>(tmw, tmx, p, splits, st);
    default: return splits > 1 ? launch_tile<256, 4, Y>(tmw, tmx, p, splits, st) : launch_wide<Y>(tmw, tmx, p, st);
  }
}

int64_t code_pitch(int64_t in_feat) { return (in_feat + 15) / 16 * 16; }

}  // namespace
}  // namespace vtq

using namespace vtq;

extern "C" {

vtq_status vtq_quantize_tokens(int32_t x_dtype, const void* x, int64_t ldx, int64_t tokens, int64_t in_feat,
                               int8_t* q, int64_t ldq, float* scale, void* stream) {
  const char* fn = "vtq_quantize_tokens";
  if (!serve_elt(x_dtype))
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (x not F32 / F16 / BF16)", fn);
  if (tokens < 0 || in_feat < 0 || tokens > INT32_MAX || ldq < in_feat)
    return serve_fail(VTQ_ERR_INTERNAL, "%s: bad shape", fn);
  if (tokens == 0) return VTQ_OK;
  if ((!x && in_feat) || (!q && in_feat) || !scale) return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null pointer", fn);
  return serve_cuda(quantize(x_dtype, x, ldx, tokens, in_feat, q, ldq, scale, static_cast<cudaStream_t>(stream)), fn);
}

size_t vtq_linear_i8_workspace_bytes(int32_t x_dtype, int64_t tokens, int64_t in_feat, int64_t out_feat) {
  (void)out_feat;
  if (x_dtype == VTQ_I8 || tokens <= 0 || in_feat < 0) return 0;
  return ((size_t)tokens * code_pitch(in_feat) + 255) / 256 * 256 + (size_t)tokens * 4;
}

vtq_status vtq_linear_i8(const vtq_linear_i8_args* a, void* ws, size_t ws_bytes, void* stream) {
  const char* fn = "vtq_linear_i8";
  if (!a) return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null arguments", fn);
  const bool codes = a->x_dtype == VTQ_I8;
  if (!codes && !serve_elt(a->x_dtype))
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (x not I8 / F32 / F16 / BF16)", fn);
  if (!serve_elt(a->y_dtype))
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (y not F32 / F16 / BF16)", fn);
  if (a->tokens < 0 || a->in_feat < 1 || a->out_feat < 0 || a->ldw < a->in_feat)
    return serve_fail(VTQ_ERR_INTERNAL, "%s: bad shape", fn);
  if (a->in_feat > kMostInputs || a->out_feat > (1 << 28) || a->tokens > (1 << 20))
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED,
                      "%s: not implemented (in_feat over 131072, out_feat over 2^28 or tokens over 2^20)", fn);
  if (a->tokens == 0 || a->out_feat == 0) return VTQ_OK;
  if (!a->x || !a->w || !a->w_scale || !a->y || (codes && !a->x_scale))
    return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null pointer", fn);
  if (!aligned16(a->w) || a->ldw % 16)
    return serve_fail(VTQ_ERR_INTERNAL, "%s: w not 16-byte aligned, or ldw not a multiple of 16", fn);
  if (codes && (!aligned16(a->x) || a->ldx % 16 || a->ldx < a->in_feat))
    return serve_fail(VTQ_ERR_INTERNAL, "%s: codes not 16-byte aligned, or ldx not a multiple of 16", fn);
  const size_t need = vtq_linear_i8_workspace_bytes(a->x_dtype, a->tokens, a->in_feat, a->out_feat);
  if (need && (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255u)))
    return serve_fail(VTQ_ERR_INVALID_ARG, "%s: workspace missing, too small or not 256-byte aligned", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int8_t* q = static_cast<const int8_t*>(a->x);
  const float* xs = a->x_scale;
  int64_t ldq = a->ldx;
  if (!codes) {
    int8_t* qw = static_cast<int8_t*>(ws);
    ldq = code_pitch(a->in_feat);
    float* sw = reinterpret_cast<float*>(qw + ((size_t)a->tokens * ldq + 255) / 256 * 256);
    if (vtq_status s = serve_cuda(quantize(a->x_dtype, a->x, a->ldx, a->tokens, a->in_feat, qw, ldq, sw, st), fn)) return s;
    q = qw;
    xs = sw;
  }
  // The smallest token tile that holds the batch; the K axis split until the CTAs fill the SMs.
  const int T = (int)a->tokens, kb = (int)((a->in_feat + 127) / 128);
  const int nt = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : T <= 128 ? 128 : 256;
  const int64_t tiles = (a->out_feat + BM - 1) / BM * ((T + nt - 1) / nt);
  // Two CTAs of a tile of up to 128 tokens fit an SM, one of 256.
  const int64_t room = (nt == 256 ? 1 : 2) * num_sms();
  const int splits = (int)std::max<int64_t>(1, std::min<int64_t>({8, room / tiles, kb / 2}));
  CUtensorMap tmw, tmx;
  cudaError_t e = tma_byte_map(&tmw, a->w, a->out_feat, a->in_feat, a->ldw, 128, BM, CU_TENSOR_MAP_SWIZZLE_128B);
  // The wide kernel's CTAs bring 128 tokens each.
  const uint32_t token_box = nt == 256 && splits == 1 ? 128 : (uint32_t)nt;
  if (e == cudaSuccess) e = tma_byte_map(&tmx, q, T, a->in_feat, ldq, 128, token_box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (e != cudaSuccess) return serve_cuda(e, fn);
  const I8Params p{T, (int)a->in_feat, (int)a->out_feat, kb, !codes, xs, a->w_scale, a->bias, a->y, a->ldy, a->status};
  if (a->y_dtype == VTQ_F32) e = product<float>(tmw, tmx, p, nt, splits, st);
  else if (a->y_dtype == VTQ_F16) e = product<__half>(tmw, tmx, p, nt, splits, st);
  else e = product<__nv_bfloat16>(tmw, tmx, p, nt, splits, st);
  return serve_cuda(e, fn);
}

}  // extern "C"
