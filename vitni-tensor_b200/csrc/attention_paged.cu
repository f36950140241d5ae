// attention_paged.cu -- attention of a batch's newest tokens over a paged key / value cache, with a
// prefix that all sequences share.
//
//   out = softmax(scale q k^T) v, one pass over the keys with the running maximum m and sum l of each
//   row's softmax:  m' = max(m, max s),  l' = l 2^(m - m') + sum 2^(s - m'),  o' likewise,
// scores in units of log2. The keys of a sequence are cut where it suits the machine; each part leaves
// (m, l, o) and attention_join_kernel adds the parts of a row.
//
// Work is a list of segments: (sequence, block of 16 query rows, kv head) over the sequence's own keys,
// then (block of 16 rows of all sequences, kv head) over the shared prefix. A row is one query head of
// one token: the heads of a kv head and the drafted tokens of a sequence fill the 16 rows of the MMA.
// The list is cut into equal runs of key tiles, one run a warp, whatever the lengths are: every CTA
// derives the same cut from the lengths on the device, so the host never needs them.
#include <algorithm>
#include <type_traits>

#include "serve.h"
#include "tc5.cuh"
#include "vtq_internal.h"

namespace vtq {

vtq_status serve_check_kv(const char* fn, const vtq_paged_kv& kv);

namespace {

constexpr int kRows = 16;      // query rows of a segment: M of the MMA
constexpr int kTileRows = 128; // of a segment of the prefix on tcgen05
constexpr int kMaxSeqs = 1024;

struct AttnParams {
  vtq_attention_args a;
  int group;        // query heads of a kv head
  int tile;         // keys of a tile
  int parts;        // warps of the whole grid
  int keys_max;     // positions that the table can hold
  int prefix;       // min(shared_len, keys_max)
  float scale_log2;
  bool q_wide;      // q rows can be read four bytes at a time
  int* plan;        // the plan arrays below, for the joining kernel
  float* part;      // slots of kRows (m, l) and o
  int dim_padded;
  // The prefix on the tensor cores' own tiles (attention_tile_kernel), where on_tiles is set:
  bool on_tiles, q_copies;           // q_copies: q rows can be copied 16 bytes at a time
  int tile_box;                      // positions of a TMA box: a page, or an even part of it; 0: none
  int tile_rt, tile_streams;         // blocks of kTileRows rows of a segment; softmax warpgroups of a CTA
  int tile_segs, tiles_each;         // segments of a kv head, steps (of tile_streams / tile_rt key tiles) of each
  int tiles_total, tile_parts;       // steps in all; CTAs that share them
  float* tile_part;                  // slots of kTileRows (m, l) and o
};

// The cut of the work: prefix sums over the sequences (index B: the shared prefix). Tiles before, and
// segments before, each sequence; its first query row; its length.
struct Plan {
  int *tiles, *segs, *q0, *len;  // [B + 2], [B + 2], [B + 1], [B + 1] (len[B]: of the prefix, 0 if nobody sees it)
};
__host__ __device__ inline int plan_ints(int B) { return 4 * (B + 2) + 2; }

__device__ __forceinline__ Plan plan_of(int* base, int B) {
  return Plan{base + 2, base + 2 + (B + 2), base + 2 + 2 * (B + 2), base + 2 + 3 * (B + 2)};
}

__device__ __forceinline__ int seq_rows(const Plan& pl, int b) { return pl.q0[b + 1] - pl.q0[b]; }

// Whether every row of a sequence sees the whole prefix. The rows of one that does not (it ends inside
// the prefix, or is empty) take no part in the prefix's segments: it has all its keys for its own, so
// that those segments need no mask for rows, and what they hold cannot reach a row that must not see it.
__device__ __forceinline__ bool sees_prefix(const AttnParams& p, const Plan& pl, int b) {
  const int n = seq_rows(pl, b);
  return n > 0 && pl.len[b] - n + 1 >= p.prefix;
}

// Built by all threads of a CTA in its shared memory; base[0] = tiles in all, base[1] = parts in use.
__device__ void build_plan(const AttnParams& p, int* base) {
  const int B = (int)p.a.kv.seqs, T = (int)p.a.tokens, H = (int)p.a.kv.kv_heads;
  const Plan pl = plan_of(base, B);
  __shared__ int s_any, s_bad, s_warp_t[32], s_warp_s[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_any = s_bad = 0;
  __syncthreads();
  for (int b = tid; b <= B; b += blockDim.x) {
    pl.q0[b] = p.a.q_start ? min(max(p.a.q_start[b], 0), T) : min(b, T);
    if (b < B) pl.len[b] = max(p.a.kv_len[b], 0);
  }
  __syncthreads();
  for (int b = tid; b < B; b += blockDim.x) {
    if (pl.q0[b + 1] < pl.q0[b]) s_bad = 1;
    else if (sees_prefix(p, pl, b)) s_any = 1;
  }
  __syncthreads();
  if (tid == 0) pl.len[B] = s_any && !s_bad ? p.prefix : 0;
  if (s_bad) {  // row starts that decrease: no sequence owns a row (the slots are counted for one owner a row)
    for (int b = tid; b <= B; b += blockDim.x) pl.q0[b] = 0;
    if (tid == 0 && p.a.status) atomicOr(p.a.status, SERVE_BAD_INDEX);
    __syncthreads();
  }
  // Inclusive sums over runs of consecutive sequences, one run a thread.
  const int n = B + 1, per = (n + (int)blockDim.x - 1) / (int)blockDim.x, b0 = min(tid * per, n), b1 = min(b0 + per, n);
  int st = 0, ss = 0;
  for (int pass = 0; pass < 2; pass++) {
    for (int b = b0; b < b1; b++) {
      int rows, keys;
      if (b < B) {
        rows = seq_rows(pl, b) * p.group;
        keys = max(min(pl.len[b], p.keys_max) - (sees_prefix(p, pl, b) ? p.prefix : 0), 0);
      } else {
        rows = p.on_tiles ? 0 : T * p.group;  // the prefix has a kernel of its own then
        keys = pl.len[B];
      }
      const int segs = (rows + kRows - 1) / kRows * H;
      if (pass) pl.tiles[b] = st, pl.segs[b] = ss;
      st += segs * ((keys + p.tile - 1) / p.tile);
      ss += segs;
    }
    if (pass == 0) {
      int it = st, is = ss;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, it, o), y = __shfl_up_sync(0xffffffffu, is, o);
        if (lane >= o) it += x, is += y;
      }
      if (lane == 31) s_warp_t[warp] = it, s_warp_s[warp] = is;
      __syncthreads();
      int ot = it - st, os = is - ss;
      for (int w = 0; w < warp; w++) ot += s_warp_t[w], os += s_warp_s[w];
      st = ot, ss = os;
    }
  }
  if (b0 < n && b1 == n) pl.tiles[n] = st, pl.segs[n] = ss;
  __syncthreads();
  if (tid == 0) {
    base[0] = pl.tiles[n];
    base[1] = min(pl.tiles[n], p.parts);
  }
  __syncthreads();
}

__device__ __forceinline__ int first_key(const AttnParams& p, const Plan& pl, int b, int B) {
  return b < B && sees_prefix(p, pl, b) ? p.prefix : 0;
}

// Part w of W covers tiles [first(w), first(w + 1)) of `total`; part_of is its inverse.
__device__ __forceinline__ int first_tile(int total, int W, int w) { return (int)((int64_t)total * w / W); }
__device__ __forceinline__ int part_of(int total, int W, int t) { return (int)((((int64_t)t + 1) * W - 1) / total); }

// Where a part stands: sequence, row block, head, tile.
struct Cursor {
  int b, mb, g, t, nt;  // nt tiles in a segment of b
  int mbs;              // row blocks of b
};

__device__ __forceinline__ int seq_tiles(const AttnParams& p, const Plan& pl, int b, int B, int* mbs) {
  const int H = (int)p.a.kv.kv_heads;
  *mbs = (pl.segs[b + 1] - pl.segs[b]) / H;
  const int segs = *mbs * H;
  return segs ? (pl.tiles[b + 1] - pl.tiles[b]) / segs : 0;
}

__device__ Cursor seek(const AttnParams& p, const Plan& pl, int B, int tile) {
  int lo = 0, hi = B;  // the last index whose tiles begin at or before `tile`
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (pl.tiles[m] <= tile) lo = m;
    else hi = m - 1;
  }
  Cursor c;
  c.b = lo;
  c.nt = seq_tiles(p, pl, lo, B, &c.mbs);
  const int at = tile - pl.tiles[lo], seg = c.nt ? at / c.nt : 0, H = (int)p.a.kv.kv_heads;
  c.t = at - seg * c.nt;
  c.mb = seg / H;
  c.g = seg - c.mb * H;
  return c;
}

// The next tile; true where it begins another segment. Never called behind the last tile.
__device__ __forceinline__ bool advance(const AttnParams& p, const Plan& pl, int B, Cursor& c) {
  if (++c.t < c.nt) return false;
  c.t = 0;
  if (++c.g == (int)p.a.kv.kv_heads) {
    c.g = 0;
    if (++c.mb == c.mbs) {
      c.mb = 0;
      do {
        c.b++;
        c.nt = c.b <= B ? seq_tiles(p, pl, c.b, B, &c.mbs) : 1;
      } while (c.b <= B && c.nt == 0);
    }
  }
  return true;
}

// The sequence that owns a row of q, or -1.
__device__ __forceinline__ int owner(const Plan& pl, int B, int token) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (pl.q0[m] <= token) lo = m;
    else hi = m - 1;
  }
  return token >= pl.q0[lo] && token < pl.q0[lo + 1] ? lo : -1;
}

template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  const int n = there ? 16 : 0;  // 0: the 16 bytes are filled with zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Whether either half of a word is an infinity or a NaN.
template <typename T>
__device__ __forceinline__ bool odd_word(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

// DP: head_dim rounded up to what the MMA loop takes (64, 128, 256). KT keys a tile, a warp's
// pipeline STAGES tiles of K and V deep; no barrier but the warp's own.
template <typename T, int DP, int KT, int WARPS, int STAGES>
__global__ void __launch_bounds__(32 * WARPS, 1) attention_part_kernel(const __grid_constant__ AttnParams p) {
  constexpr int CH = DP / 8;                         // 16-byte chunks of a row
  constexpr uint32_t kTileBytes = KT * DP * 2, kStage = 2 * kTileBytes;
  extern __shared__ __align__(128) uint8_t smem[];
  tc5::grid_release();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int B = (int)p.a.kv.seqs, H = (int)p.a.kv.kv_heads, D = (int)p.a.kv.head_dim;
  int* base = reinterpret_cast<int*>(smem + WARPS * STAGES * kStage);
  longlong2* rows = reinterpret_cast<longlong2*>(smem + WARPS * STAGES * kStage + (plan_ints(B) * 4 + 15) / 16 * 16) + warp * KT;
  __shared__ uint32_t s_valid[WARPS][STAGES];
  build_plan(p, base);
  const Plan pl = plan_of(base, B);
  const int total = base[0], W = base[1];
  if (blockIdx.x == 0) {
    for (int i = tid; i < plan_ints(B); i += blockDim.x) p.plan[i] = base[i];
    int* own = p.plan + plan_ints(B);
    for (int t = tid; t < (int)p.a.tokens; t += blockDim.x) own[t] = owner(pl, B, t);
    if (p.a.status)
      for (int b = tid; b < B; b += blockDim.x)
        if (pl.len[b] > p.keys_max || p.a.kv_len[b] < 0) atomicOr(p.a.status, SERVE_BAD_INDEX);
  }
  const int w = warp * (int)gridDim.x + (int)blockIdx.x;  // few parts spread over the SMs first
  if (w >= W) {
    tc5::grid_wait();
    return;
  }
  const int tile0 = first_tile(total, W, w), tile1 = first_tile(total, W, w + 1);
  const uint32_t stage0 = smem_u32(smem) + warp * STAGES * kStage;
  auto swizzled = [](int key, int chunk) {
    return (uint32_t)(key * DP * 2 + ((chunk ^ (key & 7)) << 4));  // eight rows' chunks in eight bank groups
  };
  const T* K = static_cast<const T*>(p.a.kv.k);
  const T* V = static_cast<const T*>(p.a.kv.v);

  // Starts tile `c` into stage s.
  auto load = [&](const Cursor& c, int s) {
    const bool shared = c.b == B;
    const int key0 = first_key(p, pl, c.b, B) + c.t * KT;
    const int end = shared ? pl.len[B] : min(pl.len[c.b], p.keys_max);
    bool ok = false;
    if (lane < KT) {
      const int pos = key0 + lane;
      int64_t ko = 0, vo = 0;
      if (pos < end) {
        const int page_size = (int)p.a.kv.page_size, at = pos / page_size;
        const int64_t page = p.a.kv.table[(pos < p.prefix ? 0 : c.b) * p.a.kv.table_ld + at], slot = pos - at * page_size;
        ok = page >= 0 && page < p.a.kv.pages;
        if (ok) {
          ko = page * p.a.kv.k_page + slot * p.a.kv.k_slot + c.g * p.a.kv.k_head;
          vo = page * p.a.kv.v_page + slot * p.a.kv.v_slot + c.g * p.a.kv.v_head;
        } else if (p.a.status) {
          atomicOr(p.a.status, SERVE_BAD_INDEX);
        }
      }
      rows[lane] = make_longlong2(ko, vo);
    }
    const uint32_t valid = __ballot_sync(0xffffffffu, ok);
    if (lane == 0) s_valid[warp][s] = valid;
    __syncwarp();
    const uint32_t k_s = stage0 + s * kStage, v_s = k_s + kTileBytes;
#pragma unroll
    for (int i = 0; i < KT * CH / 32; i++) {
      const int e = i * 32 + lane, key = e / CH, chunk = e - key * CH;
      const longlong2 o = rows[key];
      const bool there = ((valid >> key) & 1) && chunk * 8 < D;
      copy16(k_s + swizzled(key, chunk), K + (there ? o.x + chunk * 8 : 0), there);
      copy16(v_s + swizzled(key, chunk), V + (there ? o.y + chunk * 8 : 0), there);
    }
    __syncwarp();
  };

  Cursor in = seek(p, pl, B, tile0), c = in;
  int next = tile0;
  for (int s = 0; s < STAGES - 1; s++) {
    if (next < tile1) {
      load(in, s);
      if (++next < tile1) advance(p, pl, B, in);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  uint32_t qf[DP / 16][4];
  float o[DP / 8][4];
  float m0 = 0, m1 = 0, l0 = 0, l1 = 0;
  int lim0 = 0, lim1 = 0, lim_min = 0, rows_in = 0;
  bool begin = true;
  const int r0 = lane >> 2, cq = 2 * (lane & 3);
  for (int tile = tile0; tile < tile1; tile++) {
    if (begin) {
      // A new segment: its 16 query rows, and how far each of them sees.
      const bool shared = c.b == B;
      const int n = shared ? (int)p.a.tokens : seq_rows(pl, c.b), q0 = shared ? 0 : pl.q0[c.b];
      rows_in = min(kRows, n * p.group - c.mb * kRows);
      const T* qr[2];
      int lim[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int r = r0 + 8 * h, row = c.mb * kRows + r, tok = row / p.group;
        qr[h] = nullptr;
        lim[h] = 0;
        if (r < rows_in) {
          qr[h] = static_cast<const T*>(p.a.q) + (int64_t)(q0 + tok) * p.a.q_tok + (int64_t)(c.g * p.group + row - tok * p.group) * p.a.q_head;
          lim[h] = shared ? INT32_MAX : min(pl.len[c.b] - n + tok + 1, p.keys_max);
        }
      }
      lim0 = lim[0], lim1 = lim[1];
      lim_min = __reduce_min_sync(0xffffffffu, min(qr[0] ? lim0 : INT32_MAX, qr[1] ? lim1 : INT32_MAX));
#pragma unroll
      for (int k = 0; k < DP / 16; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const T* src = qr[e & 1];
          const int d = 16 * k + 8 * (e >> 1) + cq;
          uint32_t v = 0;
          if (src && d < D) {
            if (p.q_wide) {
              v = *reinterpret_cast<const uint32_t*>(src + d);
            } else {
              const uint16_t* h = reinterpret_cast<const uint16_t*>(src + d);
              v = (uint32_t)h[0] | (uint32_t)h[1] << 16;
            }
          }
          qf[k][e] = v;
        }
#pragma unroll
      for (int i = 0; i < DP / 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[i][e] = 0.0f;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.0f;
    }
    const int s = (tile - tile0) % STAGES;
    if (next < tile1) {
      load(in, (s + STAGES - 1) % STAGES);
      if (++next < tile1) advance(p, pl, B, in);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    __syncwarp();
    const uint32_t k_s = stage0 + s * kStage, v_s = k_s + kTileBytes;
    const uint32_t valid = s_valid[warp][s];
    const int key0 = first_key(p, pl, c.b, B) + c.t * KT;
    float sc[KT / 8][4];
#pragma unroll
    for (int i = 0; i < KT / 8; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) sc[i][e] = 0.0f;
#pragma unroll
    for (int k = 0; k < DP / 16; k++)
#pragma unroll
      for (int n = 0; n < KT / 16; n++) {
        uint32_t kf[4];
        const int key = 16 * n + (lane & 7) + ((lane >> 4) << 3), chunk = 2 * k + ((lane >> 3) & 1);
        ldsm4(k_s + swizzled(key, chunk), kf);
        mma16<T>(sc[2 * n], qf[k], kf[0], kf[1]);
        mma16<T>(sc[2 * n + 1], qf[k], kf[2], kf[3]);
      }
    const bool whole = valid == (KT == 32 ? 0xffffffffu : (1u << (KT & 31)) - 1u) && key0 + KT <= lim_min;
    float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < KT / 8; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int j = 8 * n + cq + e;
        sc[n][e] *= p.scale_log2;
        sc[n][2 + e] *= p.scale_log2;
        if (!whole) {
          const bool there = (valid >> j) & 1;
          if (!there || key0 + j >= lim0) sc[n][e] = -INFINITY;
          if (!there || key0 + j >= lim1) sc[n][2 + e] = -INFINITY;
        }
        x0 = fmaxf(x0, sc[n][e]);
        x1 = fmaxf(x1, sc[n][2 + e]);
      }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
    }
    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
    const float u0 = n0 == -INFINITY ? 0.0f : n0, u1 = n1 == -INFINITY ? 0.0f : n1;
    if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
      const float f0 = exp2_fast(m0 - u0), f1 = exp2_fast(m1 - u1);
      l0 *= f0, l1 *= f1;
#pragma unroll
      for (int i = 0; i < DP / 8; i++) o[i][0] *= f0, o[i][1] *= f0, o[i][2] *= f1, o[i][3] *= f1;
    }
    m0 = n0, m1 = n1;
    uint32_t pf[KT / 16][4];
#pragma unroll
    for (int n = 0; n < KT / 8; n++) {
      float e0 = exp2_fast(sc[n][0] - u0), e1 = exp2_fast(sc[n][1] - u0);
      float e2 = exp2_fast(sc[n][2] - u1), e3 = exp2_fast(sc[n][3] - u1);
      l0 += e0 + e1;
      l1 += e2 + e3;
      // The weights are rounded to the cache's type for the second product: relative to each
      // weight, so a row's error stays that of its type, as the rounding of v itself.
      pf[n >> 1][2 * (n & 1)] = pack2<T>(e0, e1);
      pf[n >> 1][2 * (n & 1) + 1] = pack2<T>(e2, e3);
    }
    if (!whole) {
      // A weight of 0 times an infinity or a NaN is no 0: values that some rows must not see are taken
      // out of the tile, and added to those that do see them.
      bool odd = false;
#pragma unroll 1
      for (int i = lane; i < KT * CH; i += 32) {
        const uint4 v = *reinterpret_cast<const uint4*>(smem + (v_s - smem_u32(smem)) + i * 16);
        odd |= odd_word<T>(v.x) || odd_word<T>(v.y) || odd_word<T>(v.z) || odd_word<T>(v.w);
      }
      if (__any_sync(0xffffffffu, odd)) {
        T* vt = reinterpret_cast<T*>(smem + (v_s - smem_u32(smem)));
#pragma unroll
        for (int i = 0; i < DP / 8; i++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int d = 8 * i + cq + e;
#pragma unroll 1
            for (int key = 0; key < KT; key++) {
              const float v = to_f32(vt[swizzled(key, d >> 3) / 2 + (d & 7)]);
              if (fabsf(v) <= 3.4028235e38f) continue;
              if (key0 + key < lim0) o[i][e] += v;
              if (key0 + key < lim1) o[i][2 + e] += v;
            }
          }
        __syncwarp();
#pragma unroll 1
        for (int i = lane; i < KT * DP; i += 32)
          if (!(fabsf(to_f32(vt[i])) <= 3.4028235e38f)) vt[i] = from_f32<T>(0.0f);
        __syncwarp();
      }
    }
#pragma unroll
    for (int k = 0; k < KT / 16; k++)
#pragma unroll
      for (int i = 0; i < DP / 16; i++) {
        uint32_t vf[4];
        const int key = 16 * k + (lane & 15), chunk = 2 * i + (lane >> 4);
        ldsm4_t(v_s + swizzled(key, chunk), vf);
        mma16<T>(o[2 * i], pf[k], vf[0], vf[1]);
        mma16<T>(o[2 * i + 1], pf[k], vf[2], vf[3]);
      }
    __syncwarp();
    const Cursor seg = c;
    begin = tile + 1 < tile1 ? advance(p, pl, B, c) : true;
    if (begin) {
      // The part's share of the segment ends here.
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
      }
      float* slot = p.part + (int64_t)(w + pl.segs[seg.b] + seg.mb * H + seg.g) * (kRows * (DP + 2));
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int r = r0 + 8 * h;
        if (r >= rows_in) continue;
        if ((lane & 3) == 0) {
          slot[2 * r] = h ? m1 : m0;
          slot[2 * r + 1] = h ? l1 : l0;
        }
        float* dst = slot + 2 * kRows + r * DP + cq;
#pragma unroll
        for (int i = 0; i < DP / 8; i++)
          *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  tc5::grid_wait();  // the join waits for this kernel alone: the prefix's has to be done with it
}

// ---- the prefix on tcgen05 ----
//
// A CTA runs STREAMS streams of one softmax warpgroup each over a run of key tiles. With RT = 2 the
// streams are two blocks of 128 query rows that share every key tile; with RT = 1 they are the even and
// the odd key tiles of one block (two parts of the same rows, joined later), so that a stream's softmax
// always runs beside the other stream's products.
//   softmax warpgroups  a thread a row: S from TMEM, the weights back into TMEM as the second product's A
//   3 loader warps      pages into a ring of swizzled K and V tiles, by TMA where a page holds 4 positions
//                       or more (gathering rows with 16-byte copies takes three warps 5700 cycles a tile,
//                       twice what the softmax needs)
//   1 warp              one thread issues S = Q K^T (N = KT keys) and O += P V (V as it lies: N-major)
// O stays in TMEM; it is scaled again only where a row's maximum has grown by more than 2^8 since the
// last time, until then the weights are taken relative to the old one (at most 256, and l with them).
// Head dims over 128 have room in TMEM for one stream; its S is double-buffered instead.

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one));
}
// N-major operand, 128-byte swizzle: 64 values of N a row of 128 bytes, 8 rows (K) an atom of 1024;
// `chunk` bytes to the next 64 values of N, 1024 to the next 8 of K.
__device__ __forceinline__ uint64_t desc_n_major(uint32_t saddr, uint32_t chunk) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | (uint64_t)(chunk >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(u[0]),
      "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
      "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]),
      "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]),
      "r"(u[29]), "r"(u[30]), "r"(u[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(u[0]),
      "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
      "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(addr)
      : "memory");
}
// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T, int DP, int KT, int RT, int STREAMS, int NSLOT>
struct TileShape {
  static constexpr uint32_t Q_TILE = kTileRows * DP * 2, Q_BYTES = RT * Q_TILE, SLOT = KT * DP * 2;
  static constexpr int THREADS = STREAMS * 128 + 128;
  static constexpr size_t SMEM = Q_BYTES + NSLOT * SLOT + 1024;
};
constexpr int kLoaders = 3, kMasks = 8;
static_assert(2 * kMasks > 8 + 1, "a mask's place must not come round before its tile's V slot has");

template <typename T, int DP, int KT, int RT, int STREAMS, int NSLOT>
__global__ void __launch_bounds__(TileShape<T, DP, KT, RT, STREAMS, NSLOT>::THREADS, 1)
    attention_tile_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap tmk,
                          const __grid_constant__ CUtensorMap tmv) {
  using L = TileShape<T, DP, KT, RT, STREAMS, NSLOT>;
  constexpr uint32_t kFmt = std::is_same<T, __half>::value ? 0u : 1u;
  constexpr uint32_t kIdescS = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((uint32_t)(KT >> 3) << 17) | (8u << 24);
  constexpr uint32_t kIdescO = (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | (8u << 24);
  constexpr int TPS = STREAMS / RT;   // key tiles of a step: 2 where the streams are the tiles
  constexpr uint32_t kColO = 2 * KT;  // columns: S / P twice, then each stream's O
  constexpr int kGroups = KT / 4;     // of 4 keys: loader lw copies groups lw, lw + 3, ..
  static_assert(2 * KT + STREAMS * DP <= 512 && NSLOT <= 8 && RT <= STREAMS, "TMEM, masks");
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_bar[2 * NSLOT + 8 + kMasks];
  __shared__ uint32_t s_valid[kMasks][kLoaders][2];
  __shared__ uint32_t s_slot;
  __shared__ int s_abort, s_any;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, ring = base + L::Q_BYTES;
  uint8_t* gbase = smem_raw + (base - smem_u32(smem_raw));
  auto bar = [&](int i) { return smem_u32(&s_bar[i]); };
  auto FULL = [&](int s) { return bar(s); };
  auto EMPTY = [&](int s) { return bar(NSLOT + s); };
  auto S_FULL = [&](int s) { return bar(2 * NSLOT + s); };      // of an S buffer: a stream's, or tile parity
  auto P_FULL = [&](int s) { return bar(2 * NSLOT + 2 + s); };
  auto PV_DONE = [&](int r) { return bar(2 * NSLOT + 4 + r); };  // of a stream
  const uint32_t Q_FULL = bar(2 * NSLOT + 6), Q_EMPTY = bar(2 * NSLOT + 7);
  auto MASK = [&](int i) { return bar(2 * NSLOT + 8 + i); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int B = (int)p.a.kv.seqs, D = (int)p.a.kv.head_dim;
  volatile int* abort_flag = &s_abort;

  tc5::grid_release();
  if (tid == 0) {
    for (int s = 0; s < NSLOT; s++) {
      tc5::bar_init(FULL(s), 32 * kLoaders);
      tc5::bar_init(EMPTY(s), 1);
    }
    for (int s = 0; s < 2; s++) {
      tc5::bar_init(S_FULL(s), 1);
      tc5::bar_init(P_FULL(s), 128);
      tc5::bar_init(PV_DONE(s), 1);
    }
    tc5::bar_init(Q_FULL, 32 * kLoaders);
    tc5::bar_init(Q_EMPTY, 1);
    for (int i = 0; i < kMasks; i++) tc5::bar_init(MASK(i), kLoaders);
    *abort_flag = 0;
    s_any = 0;
    fence_mbar_init();
  }
  constexpr int kMmaWarp = 4 * STREAMS + kLoaders;
  if (warp == kMmaWarp) tc5::alloc(smem_u32(&s_slot), 512);
  __syncthreads();
  // Nothing to do where no sequence sees the prefix (its pages need not exist then).
  for (int b = tid; b < B; b += L::THREADS) {
    const int n = (int)p.a.tokens;
    const int q0 = p.a.q_start ? min(max(p.a.q_start[b], 0), n) : b, q1 = p.a.q_start ? min(max(p.a.q_start[b + 1], 0), n) : b + 1;
    if (q1 > q0 && p.a.kv_len[b] - (q1 - q0) + 1 >= p.prefix) s_any = 1;
  }
  tc5::fence_before();
  __syncthreads();
  tc5::fence_after();
  const uint32_t tmem = s_slot;
  // Steps [step0, step1) of all segments; a segment is (kv head g, block of RT x 128 rows).
  const int step0 = first_tile(p.tiles_total, p.tile_parts, (int)blockIdx.x);
  const int steps = s_any ? first_tile(p.tiles_total, p.tile_parts, (int)blockIdx.x + 1) - step0 : 0;
  const int each = p.tiles_each, rows = (int)p.a.tokens * p.group;
  auto fail = [&]() {
    if (p.a.status) atomicOr(p.a.status, KERR_TIMEOUT);
    *abort_flag = 1;
  };
  // Whether stream r has rows in a segment.
  auto live = [&](int seg, int r) { return RT == 1 || ((seg % p.tile_segs) * RT + r) * kTileRows < rows; };
  // Bytes into a K, V or Q tile of `n` rows: blocks of 64 values, 128-byte rows, 16-byte chunks swizzled.
  auto place = [](int n, int row, int chunk) {
    return (uint32_t)((chunk >> 3) * n * 128 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
  };

  if (warp >= 4 * STREAMS) {
    if (warp < kMmaWarp) {
      // ---- loaders: tile n of this CTA in ring places 2 n (K) and 2 n + 1 (V); 8 lanes a row of 128 bytes ----
      const int lw = warp - 4 * STREAMS, sub = lane >> 3;
      const T* K = static_cast<const T*>(p.a.kv.k);
      const T* V = static_cast<const T*>(p.a.kv.v);
      const int page_size = (int)p.a.kv.page_size;
      const int box = p.tile_box, boxes = box ? KT / box : 0;  // keys of a TMA box, boxes of a tile (32 at most)
      int told = 0;  // ring places that the consumers have been told of
      auto tell = [&](int upto) {  // the copies of every place before `upto` have landed
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        for (; told < upto; told++) tc5::bar_arrive(FULL(told % NSLOT));
      };
      // This lane's two keys of a tile (rows 32 h + lane of those that this warp copies).
      auto key_of = [&](int h) {
        const int k = 32 * h + lane, grp = lw + kLoaders * (k >> 2);
        return grp < kGroups ? 4 * grp + (k & 3) : -1;
      };
      const int key_a = key_of(0), key_b = key_of(1);
      // The page of a position; -1 behind the prefix.
      auto page_at = [&](int pos) { return pos < p.prefix ? p.a.kv.table[pos / page_size] : -1; };
      int seg = step0 / each, kt = (step0 - seg * each) * TPS;
      int g = seg / p.tile_segs;
      bool new_seg = true;
      int segs_seen = 0;
      const int tiles = steps * TPS;
      bool ok = true;
      // Waits until ring place n may be filled; meanwhile tells of whatever has landed.
      auto claim = [&](int n) {
        if (n < NSLOT) return true;
        const uint32_t ph = tc5::phase(n, NSLOT, true);
        if (!tc5::bar_try(EMPTY(n % NSLOT), ph)) {
          if (told < n) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            tell(n);
          }
          if (!tc5::bar_wait(EMPTY(n % NSLOT), ph)) return false;
        }
        return true;
      };
      // The page of this lane's box of the next tile, read a tile ahead.
      int box_page = lane < boxes && steps ? page_at(kt * KT + lane * box) : -1;
      for (int n = 0; n < tiles && ok && !*abort_flag; n++) {
        const bool with_q = new_seg;
        if (new_seg) {
          if (segs_seen) {
            // The products with the Q before need every tile so far.
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            tell(2 * n);
            if (!tc5::bar_wait(Q_EMPTY, tc5::phase(segs_seen - 1, 1))) {
              ok = false;
              break;
            }
          }
          segs_seen++;
          new_seg = false;
          const int row0 = (seg - g * p.tile_segs) * RT * kTileRows;
#pragma unroll 1
          for (int r = lw * 4 + sub; r < RT * kTileRows; r += 4 * kLoaders) {
            const int row = row0 + r, tok = row / p.group;
            const bool in = row < rows;
            const T* src = static_cast<const T*>(p.a.q) + (in ? (int64_t)tok * p.a.q_tok + (int64_t)(g * p.group + row - tok * p.group) * p.a.q_head : 0);
#pragma unroll
            for (int c = 0; c < DP / 64; c++) {
              const int chunk = c * 8 + (lane & 7);
              const bool there = in && chunk * 8 < D;
              const uint32_t at = (r / kTileRows) * L::Q_TILE + place(kTileRows, r % kTileRows, chunk);
              if (p.q_copies) {
                copy16(base + at, src + (there ? chunk * 8 : 0), there);
              } else {
                T* dst = reinterpret_cast<T*>(gbase + at);
#pragma unroll
                for (int e = 0; e < 8; e++) dst[e] = there ? src[chunk * 8 + e] : from_f32<T>(0.0f);
              }
            }
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          __syncwarp();
        }
        const uint32_t k_s = ring + (2 * n % NSLOT) * L::SLOT, v_s = ring + ((2 * n + 1) % NSLOT) * L::SLOT;
        // A tile that lies whole in pages that exist comes by TMA, a box for each page (or piece of one):
        // every loader warp sees the same pages and takes the same way. The prefix's last tile, one with a
        // bad page, and pages of fewer than 4 positions are gathered row by row, zeros in the gaps (what
        // lies behind the prefix in its last page may be anything, and 0 times NaN is no 0).
        const int box_pos = kt * KT + lane * box;
        const bool by_box = boxes && !__any_sync(0xffffffffu, lane < boxes && (box_page < 0 || box_page >= p.a.kv.pages || box_pos + box > p.prefix));
        const int this_kt = kt, this_g = g, this_page = box_page;
        if (++kt == each * TPS) {
          kt = 0;
          new_seg = true;
          if (++seg, seg % p.tile_segs == 0) g++;
        }
        if (lane < boxes && n + 1 < tiles) box_page = page_at(kt * KT + lane * box);
        if (by_box) {
          if (told < 2 * n) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            tell(2 * n);
          }
#pragma unroll 1
          for (int h = 0; h < 2 && ok; h++) {
            ok = claim(2 * n + h);
            __syncwarp();
            if (!ok) break;
            if (h == 0 && lane == 0) {
#pragma unroll
              for (int w = 0; w < 2; w++) {
                const int keys = 4 * ((kGroups - lw + kLoaders - 1) / kLoaders) - 32 * w;
                s_valid[n % kMasks][lw][w] = keys >= 32 ? 0xffffffffu : keys > 0 ? (1u << keys) - 1u : 0u;
              }
              tc5::bar_arrive(MASK(n % kMasks));
            }
            const uint32_t full = FULL((2 * n + h) % NSLOT);
            if (lw == h && lane == 0) tc5::bar_expect(full, L::SLOT);
            else tc5::bar_arrive(full);
            told = 2 * n + h + 1;
            __syncwarp();
            if (lw == h && lane < boxes) {
              const uint32_t dst = (h ? v_s : k_s) + lane * box * 128;
              const int slot = box_pos % page_size;
#pragma unroll
              for (int c = 0; c < DP / 64; c++) tc5::tma_4d(dst + c * KT * 128, h ? &tmv : &tmk, 64 * c, slot, this_g, this_page, full);
            }
          }
        } else {
          // Offsets of this lane's keys.
          int64_t ka = 0, va = 0, kb = 0, vb = 0;
          auto offsets = [&](int key, int64_t& ko, int64_t& vo) {
            const int pos = this_kt * KT + key;
            if (key < 0 || pos >= p.prefix) return false;
            const int page = page_at(pos);
            if (page < 0 || page >= p.a.kv.pages) {
              if (p.a.status) atomicOr(p.a.status, SERVE_BAD_INDEX);
              return false;
            }
            const int64_t slot = pos % page_size;
            ko = page * p.a.kv.k_page + slot * p.a.kv.k_slot + this_g * p.a.kv.k_head;
            vo = page * p.a.kv.v_page + slot * p.a.kv.v_slot + this_g * p.a.kv.v_head;
            return true;
          };
          const uint32_t in_a = __ballot_sync(0xffffffffu, offsets(key_a, ka, va));
          const uint32_t in_b = __ballot_sync(0xffffffffu, offsets(key_b, kb, vb));
#pragma unroll 1
          for (int h = 0; h < 2 && ok; h++) {
            ok = claim(2 * n + h);
            __syncwarp();
            if (!ok) break;
            if (h == 0 && lane == 0) {
              s_valid[n % kMasks][lw][0] = in_a;
              s_valid[n % kMasks][lw][1] = in_b;
              tc5::bar_arrive(MASK(n % kMasks));
            }
            const T* from = h ? V : K;
            const int64_t oa = h ? va : ka, ob = h ? vb : kb;
            const uint32_t dst = h ? v_s : k_s;
#pragma unroll 4
            for (int i = 0; i < (kGroups + kLoaders - 1) / kLoaders; i++) {
              const int grp = lw + kLoaders * i, src = (4 * i + sub) & 31;
              const int64_t o = __shfl_sync(0xffffffffu, i < 8 ? oa : ob, src);
              const bool in = ((i < 8 ? in_a : in_b) >> src) & 1;
              if (grp < kGroups) {
#pragma unroll
                for (int c = 0; c < DP / 64; c++) {
                  const int chunk = c * 8 + (lane & 7);
                  const bool there = in && chunk * 8 < D;
                  copy16(dst + place(KT, 4 * grp + sub, chunk), from + (there ? o + chunk * 8 : 0), there);
                }
              }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
          }
          if (!ok) break;
          asm volatile("cp.async.wait_group 2;" ::: "memory");
          if (told < 2 * n) tell(2 * n);
        }
        if (with_q) {
          if (by_box) asm volatile("cp.async.wait_group 0;" ::: "memory");
          else asm volatile("cp.async.wait_group 2;" ::: "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          tc5::bar_arrive(Q_FULL);
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      if (ok && !*abort_flag) tell(2 * tiles);
      else if (lane == 0) fail();
    } else {
      // ---- products ----
      const uint32_t one = tc5::elect();
      int segs_seen = 0;
      bool ok = true;
      // S of step i for stream r: its key tile is n. `seg_of` and `in_of`: the segment of a step and the
      // step's place in it, for this step and the next (divisions are slow next to an MMA).
      int seg_of[2], in_of[2];
      seg_of[0] = step0 / each;
      in_of[0] = step0 - seg_of[0] * each;
      auto follow = [&]() {
        in_of[1] = in_of[0] + 1 == each ? 0 : in_of[0] + 1;
        seg_of[1] = seg_of[0] + (in_of[1] == 0);
      };
      follow();
      auto first = [&](int i, int r, int k_) {
        const int n = i * TPS + (TPS == 2 ? r : 0), buf = STREAMS == 2 ? r : (n & 1), at = 2 * n % NSLOT;
        const int in = in_of[k_];
        if (r == 0 && (i == 0 || in == 0)) {
          if (!tc5::bar_wait(Q_FULL, tc5::phase(segs_seen, 1))) return false;
          segs_seen++;
        }
        if ((TPS == 2 || r == 0) && !tc5::bar_wait(FULL(at), tc5::phase(2 * n, NSLOT))) return false;
        tc5::fence_after();
        const bool on = live(seg_of[k_], r);
        const uint32_t qs = base + (RT == 2 ? r : 0) * L::Q_TILE, ks = ring + at * L::SLOT;
        if (on) {
#pragma unroll
          for (int k = 0; k < DP / 16; k++)
            mma_ss(tmem + buf * KT, tc5::desc_sw128(qs + (k >> 2) * (kTileRows * 128) + (k & 3) * 32),
                   tc5::desc_sw128(ks + (k >> 2) * (KT * 128) + (k & 3) * 32), kIdescS, k > 0, one);
          tc5::commit(S_FULL(buf), one);
        }
        if (TPS == 2 || r == RT - 1) tc5::commit(EMPTY(at), one);
        if (r == STREAMS - 1 && (i + 1 == steps || in + 1 == each)) tc5::commit(Q_EMPTY, one);
        return true;
      };
      // O of stream r += P V at step i; u: how many P the buffer has had.
      int used[2] = {0, 0};
      auto second = [&](int i, int r) {
        const int n = i * TPS + (TPS == 2 ? r : 0), buf = STREAMS == 2 ? r : (n & 1), at = (2 * n + 1) % NSLOT;
        const bool on = live(seg_of[0], r);
        if (on && !tc5::bar_wait(P_FULL(buf), used[buf]++ & 1)) return false;
        if ((TPS == 2 || r == 0) && !tc5::bar_wait(FULL(at), tc5::phase(2 * n + 1, NSLOT))) return false;
        tc5::fence_after();
        const bool start = i == 0 || in_of[0] == 0;
        const uint32_t vs = ring + at * L::SLOT;
        if (on) {
#pragma unroll
          for (int k = 0; k < KT / 16; k++)
            mma_ts(tmem + kColO + r * DP, tmem + buf * KT + 8 * k, desc_n_major(vs + k * 2048, KT * 128), kIdescO, !start || k > 0, one);
          tc5::commit(PV_DONE(r), one);
        }
        if (TPS == 2 || r == RT - 1) tc5::commit(EMPTY(at), one);
        return true;
      };
      if (steps) {
        for (int r = 0; r < STREAMS && ok; r++) ok = first(0, r, 0);
        for (int i = 0; i < steps && ok; i++) {
#pragma unroll
          for (int r = 0; r < STREAMS; r++) {
            if constexpr (STREAMS == 1) {
              ok = (i + 1 == steps || first(i + 1, 0, 1)) && second(i, 0);
            } else {
              ok = ok && second(i, r) && (i + 1 == steps || first(i + 1, r, 1));
            }
          }
          seg_of[0] = seg_of[1];
          in_of[0] = in_of[1];
          follow();
        }
      }
      if (!ok && lane == 0) fail();
    }
  } else {
    // ---- softmax: row `row` of stream r ----
    const int r = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, so = tmem + lanes + kColO + r * DP;
    float m = -INFINITY, l = 0.0f;  // m: what the weights are relative to
    int used = 0;                   // tiles that this stream has had
    int seg = step0 / each, in = step0 - seg * each;
    for (int i = 0; i < steps; i++) {
      const bool start = i == 0 || in == 0, last = i + 1 == steps || in + 1 == each;
      const int this_seg = seg;
      if (++in == each) in = 0, seg++;
      if (!live(this_seg, r)) continue;
      const int n = i * TPS + (TPS == 2 ? r : 0), buf = STREAMS == 2 ? r : (n & 1);
      const uint32_t sp = tmem + lanes + buf * KT;
      bool whole = tc5::bar_wait(MASK(n % kMasks), tc5::phase(n, kMasks));
      if (!whole || !tc5::bar_wait(S_FULL(buf), (STREAMS == 2 ? used : used >> 1) & 1)) {
        if (lane == 0) fail();
        break;
      }
      tc5::fence_after();
      // The row is read twice, 32 columns at a time, in loops that stay in the instruction cache: the same
      // arithmetic unrolled over a whole row waits more for instructions than for anything else (2.4 of
      // 4 cycles an instruction, 86 us on 64 sequences behind 32768 keys).
#pragma unroll
      for (int w = 0; w < kLoaders; w++) {
        const int keys = 4 * ((kGroups - w + kLoaders - 1) / kLoaders);
        const uint32_t lo = keys >= 32 ? 0xffffffffu : (1u << (keys & 31)) - 1u, hi = keys > 32 ? (1u << (keys - 32)) - 1u : 0u;
        whole = whole && s_valid[n % kMasks][w][0] == lo && s_valid[n % kMasks][w][1] == hi;
      }
      if (!whole) {
        // The prefix's end, or a page that does not exist: those scores become what no other can exceed.
        const float never = p.scale_log2 > 0.0f ? -INFINITY : INFINITY;
#pragma unroll 1
        for (int c = 0; c < KT / 32; c++) {
          float x[32];
          tmem_ld32(sp + 32 * c, x);
          tc5::wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j++) {
            const int grp = 8 * c + (j >> 2), w = grp % kLoaders, k = 4 * (grp / kLoaders) + (j & 3);
            if (!((s_valid[n % kMasks][w][k >> 5] >> (k & 31)) & 1)) x[j] = never;
          }
          tmem_st32(sp + 32 * c, reinterpret_cast<const uint32_t*>(x));
        }
        tmem_wait_st();
      }
      float top;
      if (p.scale_log2 > 0.0f) {
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < KT / 64; c++) {
          float x[64];
          tmem_ld32(sp + 64 * c, x);
          tmem_ld32(sp + 64 * c + 32, x + 32);
          tc5::wait_ld();
          float a = fmaxf(x[0], x[1]), b = fmaxf(x[2], x[3]);
#pragma unroll
          for (int j = 4; j < 64; j += 4) {
            t0 = fmaxf(fmaxf(x[j], x[j + 1]), t0);
            t1 = fmaxf(fmaxf(x[j + 2], x[j + 3]), t1);
          }
          t0 = fmaxf(t0, a);
          t1 = fmaxf(t1, b);
        }
        top = fmaxf(t0, t1) * p.scale_log2;
      } else {  // the largest score is that of the smallest product
        float low = INFINITY;
#pragma unroll 1
        for (int c = 0; c < KT / 32; c++) {
          float x[32];
          tmem_ld32(sp + 32 * c, x);
          tc5::wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j++) low = fminf(low, x[j]);
        }
        top = low * p.scale_log2;
      }
      if (start) {
        m = top;
        l = 0.0f;
      } else {
        const bool grow = top > m + 8.0f || (m == -INFINITY && top > -INFINITY);
        if (__any_sync(0xffffffffu, grow)) {
          const float to = grow ? top : m;
          const float f = !grow ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(m - to);
          if (!tc5::bar_wait(PV_DONE(r), (used - 1) & 1)) {
            if (lane == 0) fail();
            break;
          }
          tc5::fence_after();
#pragma unroll 1
          for (int c = 0; c < DP / 32; c++) {
            float o[32];
            tmem_ld32(so + 32 * c, o);
            tc5::wait_ld();
#pragma unroll
            for (int j = 0; j < 32; j++) o[j] *= f;
            tmem_st32(so + 32 * c, reinterpret_cast<const uint32_t*>(o));
          }
          tmem_wait_st();
          l *= f;
          m = to;
        }
      }
      const float u = m == -INFINITY ? 0.0f : m;
      // P in the place of S: 16 columns for 32, so that a chunk never lands on columns not read yet.
      const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), u2 = make_float2(-u, -u);
      float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
      float x[32];
      tmem_ld32(sp, x);
#pragma unroll 1
      for (int c = 0; c < KT / 32; c++) {
        tc5::wait_ld();
        float2 e[16];
#pragma unroll
        for (int j = 0; j < 16; j++) e[j] = fma2(make_float2(x[2 * j], x[2 * j + 1]), scale2, u2);
        if (c + 1 < KT / 32) tmem_ld32(sp + 32 * (c + 1), x);
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 16; j++) {
          e[j].x = exp2_fast(e[j].x);
          e[j].y = exp2_fast(e[j].y);
          if (j & 1) sum1 = add2(sum1, e[j]);
          else sum0 = add2(sum0, e[j]);
          w[j] = pack2<T>(e[j].x, e[j].y);
        }
        tmem_st16(sp + 16 * c, w);
      }
      l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
      tmem_wait_st();
      tc5::fence_before();
      tc5::bar_arrive(P_FULL(buf));
      used++;
      if (last) {
        if (!tc5::bar_wait(PV_DONE(r), (used - 1) & 1)) {
          if (lane == 0) fail();
          break;
        }
        tc5::fence_after();
        float* slot = p.tile_part + (int64_t)(((int)blockIdx.x + this_seg) * STREAMS + r) * (kTileRows * (DP + 2));
        const bool there = ((this_seg % p.tile_segs) * RT + (RT == 2 ? r : 0)) * kTileRows + row < rows;
        if (there) *reinterpret_cast<float2*>(slot + 2 * row) = make_float2(m, l);
#pragma unroll 1
        for (int c = 0; c < DP / 32; c++) {
          float o[32];
          tmem_ld32(so + 32 * c, o);
          tc5::wait_ld();
          if (there) {
            float4* dst = reinterpret_cast<float4*>(slot + 2 * kTileRows + row * DP + 32 * c);
#pragma unroll
            for (int j = 0; j < 8; j++) dst[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          }
        }
        tc5::fence_before();
      }
    }
  }
  tc5::fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc5::fence_after();
    tc5::dealloc(tmem, 512);
  }
}

// Adds the parts of each row (query head of a token): one warp a row.
template <typename T, int DP>
__global__ void __launch_bounds__(128) attention_join_kernel(const __grid_constant__ AttnParams p) {
  tc5::grid_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int heads = (int)p.a.heads, H = (int)p.a.kv.kv_heads, B = (int)p.a.kv.seqs, D = (int)p.a.kv.head_dim;
  if (row >= p.a.tokens * heads) return;
  const int token = (int)(row / heads), head = (int)(row - (int64_t)token * heads), g = head / p.group;
  const Plan pl = plan_of(p.plan, B);
  const int b = p.plan[plan_ints(B) + token];
  if (b < 0) return;  // no sequence owns the row
  const int total = p.plan[0], W = p.plan[1];
  // The row's place among the sequence's own rows, and among all rows for the prefix.
  int count[2], rr[2];
  const float* slot0[2];
  const bool with_prefix = sees_prefix(p, pl, b) && p.prefix > 0;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const int s = k ? B : b, r = (k ? token : token - pl.q0[b]) * p.group + head - g * p.group;
    count[k] = rr[k] = 0;
    slot0[k] = nullptr;
    if (k && !with_prefix) continue;
    if (k && p.on_tiles) {
      // A CTA leaves a part for each stream: of other rows, or of the same rows' other keys.
      const int mt = r / (kTileRows * p.tile_rt), seg = g * p.tile_segs + mt, w = part_of(p.tiles_total, p.tile_parts, seg * p.tiles_each);
      const int in = r - mt * kTileRows * p.tile_rt, stream = in / kTileRows;
      rr[k] = in - stream * kTileRows;
      count[k] = (part_of(p.tiles_total, p.tile_parts, (seg + 1) * p.tiles_each - 1) - w + 1) * (p.tile_streams / p.tile_rt);
      slot0[k] = p.tile_part + ((int64_t)(w + seg) * p.tile_streams + stream) * (kTileRows * (DP + 2));
      continue;
    }
    const int mb = r / kRows;
    int mbs;
    const int nt = seq_tiles(p, pl, s, B, &mbs);
    if (!nt) continue;
    const int t0 = pl.tiles[s] + (mb * H + g) * nt, w = part_of(total, W, t0);
    rr[k] = r - mb * kRows;
    count[k] = part_of(total, W, t0 + nt - 1) - w + 1;
    slot0[k] = p.part + (int64_t)(w + pl.segs[s] + mb * H + g) * (kRows * (DP + 2));
  }
  const int parts = count[0] + count[1];
  // Part i's (m, l) of the row, and its o.
  auto at = [&](int i, const float*& o) {
    const int k = i >= count[0], rows = k && p.on_tiles ? kTileRows : kRows;
    const int step = rows * (DP + 2) * (k && p.on_tiles ? p.tile_rt : 1);
    const float* s = slot0[k] + (int64_t)(i - (k ? count[0] : 0)) * step;
    o = s + 2 * rows + rr[k] * DP;
    return s + 2 * rr[k];
  };
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 32) {
    const float* o;
    m = fmaxf(m, *at(i, o));
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  const float um = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, acc[DP / 32];
#pragma unroll
  for (int e = 0; e < DP / 32; e++) acc[e] = 0.0f;
  for (int i0 = 0; i0 < parts; i0 += 32) {
    float f = 0.0f;
    if (i0 + lane < parts) {
      const float* o;
      const float2 ml = *reinterpret_cast<const float2*>(at(i0 + lane, o));
      f = exp2_fast(ml.x - um);
      l += f * ml.y;
    }
    const int n = min(32, parts - i0);
#pragma unroll 4
    for (int i = 0; i < n; i++) {
      const float* s;
      at(i0 + i, s);
      const float fi = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
      for (int e = 0; e < DP / 32; e++) acc[e] = fmaf(fi, s[lane + 32 * e], acc[e]);
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key: zeros
  T* out = static_cast<T*>(p.a.out) + token * p.a.o_tok + head * p.a.o_head;
#pragma unroll
  for (int e = 0; e < DP / 32; e++)
    if (lane + 32 * e < D) out[lane + 32 * e] = from_f32<T>(acc[e] * inv);
  if (p.a.lse && lane == 0)
    p.a.lse[token * p.a.lse_tok + head] = l == 0.0f ? -INFINITY : (um + log2f(l)) * 0.69314718055994531f;
}

int padded_dim(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
int part_warps(int dp) { return dp == 256 ? 4 : 8; }

// How the prefix goes to the tensor cores' own tiles, and where: more rows than the 16 that one read of
// a key serves in the part kernel, and keys enough to pay for another launch.
struct TileCut {
  bool on;
  int keys, rt, streams, segs, each;  // keys of a tile; see AttnParams
  int64_t total;
};
TileCut tile_cut(const vtq_attention_args& a) {
  TileCut c = {};
  const int64_t rows = a.tokens * (a.heads / a.kv.kv_heads), prefix = std::min(a.shared_len, a.kv.table_width * a.kv.page_size);
  c.on = rows > 16 && prefix >= 512;
  const bool wide = a.kv.head_dim > 128;
  c.keys = wide ? 64 : 128;
  c.streams = wide ? 1 : 2;
  c.rt = !wide && rows > kTileRows ? 2 : 1;
  c.segs = (int)((rows + kTileRows * c.rt - 1) / (kTileRows * c.rt));
  const int step = c.keys * c.streams / c.rt;
  c.each = (int)((prefix + step - 1) / step);
  c.total = a.kv.kv_heads * (int64_t)c.segs * c.each;
  return c;
}
size_t tile_bytes(const vtq_attention_args& a) {
  const TileCut c = tile_cut(a);
  if (!c.on) return 0;
  const int64_t slots = (std::min<int64_t>(c.total, num_sms()) + a.kv.kv_heads * c.segs) * c.streams;
  return (size_t)slots * kTileRows * (padded_dim(a.kv.head_dim) + 2) * 4;
}

size_t plan_bytes(const vtq_attention_args& a) {
  return ((size_t)(plan_ints((int)a.kv.seqs) + a.tokens) * 4 + 255) / 256 * 256;
}
// Segments of any lengths: each sequence's rows and, once more, all rows for the prefix.
int64_t most_segments(const vtq_attention_args& a) {
  const int64_t group = a.heads / a.kv.kv_heads, rows = a.tokens * group;
  return (rows / kRows + a.kv.seqs + (a.shared_len && !tile_cut(a).on ? (rows + kRows - 1) / kRows : 0)) * a.kv.kv_heads;
}

size_t part_bytes(const vtq_attention_args& a) {
  const int dp = padded_dim(a.kv.head_dim);
  const int64_t slots = most_segments(a) + (int64_t)num_sms() * part_warps(dp);
  return ((size_t)slots * kRows * (dp + 2) * 4 + 255) / 256 * 256;
}

vtq_status check(const char* fn, const vtq_attention_args* a) {
  if (!a) return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null arguments", fn);
  if (vtq_status s = serve_check_kv(fn, a->kv)) return s;
  if (a->tokens < 0 || a->heads < 1 || a->heads % a->kv.kv_heads || a->shared_len < 0)
    return serve_fail(VTQ_ERR_INTERNAL, "%s: bad shape (heads not a multiple of kv_heads, or a negative size)", fn);
  if (a->kv.seqs > kMaxSeqs)
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (over %d sequences in one call)", fn, kMaxSeqs);
  if (a->tokens > (1 << 20) || a->heads > 65536 || a->kv.table_width * a->kv.page_size > INT32_MAX / 2)
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (over 2^20 tokens, 2^16 heads or 2^30 positions)", fn);
  const int64_t tiles = (a->kv.table_width * a->kv.page_size + 15) / 16 + 1;
  if (most_segments(*a) * tiles > INT32_MAX || tile_cut(*a).total > INT32_MAX)
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (query rows times table positions over 2^35)", fn);
  return VTQ_OK;
}

template <typename T, int DP, int KT, int RT, int STREAMS, int NSLOT>
cudaError_t launch_tiles(const AttnParams& p, cudaStream_t st) {
  using L = TileShape<T, DP, KT, RT, STREAMS, NSLOT>;
  auto tiles = attention_tile_kernel<T, DP, KT, RT, STREAMS, NSLOT>;
  const cudaError_t e = cudaFuncSetAttribute(tiles, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::SMEM);
  if (e != cudaSuccess) return e;
  // A box is the largest power of two of positions that pages are made of.
  AttnParams q = p;
  CUtensorMap tmk = {}, tmv = {};
  const vtq_paged_kv& kv = p.a.kv;
  q.tile_box = 1;
  while (q.tile_box < KT && kv.page_size % (2 * q.tile_box) == 0) q.tile_box *= 2;
  if (KT / q.tile_box > 32) {
    q.tile_box = 0;
  } else {
    const uint64_t dim[4] = {(uint64_t)kv.head_dim, (uint64_t)kv.page_size, (uint64_t)kv.kv_heads, (uint64_t)kv.pages};
    const uint64_t ks[3] = {2 * (uint64_t)kv.k_slot, 2 * (uint64_t)kv.k_head, 2 * (uint64_t)kv.k_page};
    const uint64_t vs[3] = {2 * (uint64_t)kv.v_slot, 2 * (uint64_t)kv.v_head, 2 * (uint64_t)kv.v_page};
    if (tma_half_map(&tmk, kv.k, dim, ks, 64, (uint32_t)q.tile_box) != cudaSuccess ||
        tma_half_map(&tmv, kv.v, dim, vs, 64, (uint32_t)q.tile_box) != cudaSuccess)
      q.tile_box = 0;  // strides that TMA does not take: rows are gathered
  }
  kernel_launch_count()++;
  tiles<<<(unsigned)p.tile_parts, L::THREADS, L::SMEM, st>>>(q, tmk, tmv);
  return cudaGetLastError();
}

template <typename T, int DP, int KT, int WARPS, int STAGES>
cudaError_t launch(const AttnParams& p, cudaStream_t st) {
  auto part = attention_part_kernel<T, DP, KT, WARPS, STAGES>;
  const size_t smem = (size_t)WARPS * STAGES * 2 * KT * DP * 2 + (plan_ints((int)p.a.kv.seqs) * 4 + 15) / 16 * 16 +
                      (size_t)WARPS * KT * sizeof(longlong2);
  cudaError_t e = cudaFuncSetAttribute(part, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  if (p.on_tiles) {
    if constexpr (DP == 256) e = launch_tiles<T, 256, 64, 1, 1, 5>(p, st);
    else if constexpr (DP == 128) e = p.tile_rt == 2 ? launch_tiles<T, 128, 128, 2, 2, 5>(p, st) : launch_tiles<T, 128, 128, 1, 2, 6>(p, st);
    else e = p.tile_rt == 2 ? launch_tiles<T, 64, 128, 2, 2, 8>(p, st) : launch_tiles<T, 64, 128, 1, 2, 8>(p, st);
    if (e != cudaSuccess) return e;
  }
  kernel_launch_count() += 2;
  // Each waits for the one before at its own point (griddepcontrol): the part kernel at its end.
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.parts / WARPS));
  cfg.blockDim = dim3(32 * WARPS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.on_tiles && pdl_enabled() ? 1 : 0;
  if ((e = cudaLaunchKernelEx(&cfg, part, p)) != cudaSuccess) return e;
  cfg.gridDim = dim3((unsigned)((p.a.tokens * p.a.heads + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, attention_join_kernel<T, DP>, p);
}

template <typename T>
cudaError_t launch_dim(AttnParams& p, cudaStream_t st) {
  switch (p.dim_padded) {
    case 64: return launch<T, 64, 32, 8, 3>(p, st);
    case 128: return launch<T, 128, 16, 8, 3>(p, st);
    default: return launch<T, 256, 16, 4, 3>(p, st);
  }
}

}  // namespace
}  // namespace vtq

using namespace vtq;

extern "C" {

size_t vtq_attention_paged_workspace_bytes(const vtq_attention_args* a) {
  if (check("vtq_attention_paged", a) || a->tokens == 0 || a->kv.seqs == 0) return 0;
  return plan_bytes(*a) + part_bytes(*a) + tile_bytes(*a);
}

vtq_status vtq_attention_paged(const vtq_attention_args* a, void* ws, size_t ws_bytes, void* stream) {
  const char* fn = "vtq_attention_paged";
  if (vtq_status s = check(fn, a)) return s;
  if (a->tokens == 0 || a->kv.seqs == 0) return VTQ_OK;
  if (!a->q || !a->out || !a->kv_len) return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null pointer", fn);
  const size_t need = vtq_attention_paged_workspace_bytes(a);
  if (!ws || ws_bytes < need || (reinterpret_cast<uintptr_t>(ws) & 255u))
    return serve_fail(VTQ_ERR_INVALID_ARG, "%s: workspace missing, too small or not 256-byte aligned", fn);
  AttnParams p = {};
  p.a = *a;
  p.group = (int)(a->heads / a->kv.kv_heads);
  p.dim_padded = padded_dim(a->kv.head_dim);
  p.tile = p.dim_padded == 64 ? 32 : 16;
  p.parts = num_sms() * part_warps(p.dim_padded);
  p.keys_max = (int)(a->kv.table_width * a->kv.page_size);
  p.prefix = (int)std::min<int64_t>(a->shared_len, p.keys_max);
  // A scale of 0 weighs every key alike: so does one that no product reaches.
  p.scale_log2 = a->scale == 0.0f ? 1e-30f : a->scale * 1.4426950408889634f;
  p.q_wide = (reinterpret_cast<uintptr_t>(a->q) & 3u) == 0 && a->q_tok % 2 == 0 && a->q_head % 2 == 0;
  p.plan = static_cast<int*>(ws);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + plan_bytes(*a));
  const TileCut c = tile_cut(*a);
  p.on_tiles = c.on;
  if (c.on) {
    p.q_copies = aligned16(a->q) && a->q_tok % 8 == 0 && a->q_head % 8 == 0;
    p.tile_rt = c.rt;
    p.tile_streams = c.streams;
    p.tile_segs = c.segs;
    p.tiles_each = c.each;
    p.tiles_total = (int)c.total;
    p.tile_parts = std::min(p.tiles_total, num_sms());
    p.tile_part = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.part) + part_bytes(*a));
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return serve_cuda(a->kv.dtype == VTQ_F16 ? launch_dim<__half>(p, st) : launch_dim<__nv_bfloat16>(p, st), fn);
}

}  // extern "C"
