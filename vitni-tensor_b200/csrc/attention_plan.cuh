// attention_plan.cuh -- attention_paged: parameters, the cut of the work that every CTA derives from the
// lengths on the device, and small pieces that both kinds of work use.
#pragma once
#include <type_traits>

#include "serve.h"
#include "tc5.cuh"
#include "vtq_internal.h"

namespace vtq {

namespace {

constexpr int kRows = 16;      // query rows of a segment: M of the MMA
constexpr int kTileRows = 128; // of a segment of the prefix on tcgen05
constexpr int kMaxSeqs = 1024;
constexpr int kBytesPerCycle = 3500;  // from HBM, of all SMs

// n / d for 0 <= n < 2^31, d >= 1: with 2^s >= d, m = floor(2^32 (2^s - d) / d) + 1 and (mulhi(m, n) + n) >> s.
struct Divisor {
  uint32_t mul;
  int shift;
  __host__ __device__ __forceinline__ int operator()(int n) const {
#ifdef __CUDA_ARCH__
    const uint32_t high = __umulhi(mul, (uint32_t)n);
#else
    const uint32_t high = (uint32_t)((uint64_t)mul * (uint32_t)n >> 32);
#endif
    return (int)((high + (uint32_t)n) >> shift);
  }
};
inline Divisor divisor(int64_t d) {
  int s = 0;
  while ((1ll << s) < d) s++;
  return Divisor{(uint32_t)((((uint64_t)((1ll << s) - d)) << 32) / (uint64_t)d + 1), s};
}

// What the two kinds of work take of an SM, in cycles (measured; attention_paged.cu).
struct Costs {
  int tile, segment, begin;   // a part's tile, a segment of parts, and what passes before and behind them
  int step, tile_segment;     // a step of the prefix's own tiles, and a segment of them
  int tile_bytes;             // of a part's tile, from HBM
};

struct AttnParams {
  vtq_attention_args a;
  int group;        // query heads of a kv head
  int tile;         // keys of a part's tile, a power of two,
  int tile_shift;   // and which
  Divisor by_page, by_group;
  int ctas, warps;  // of the grid; warps of a CTA that take parts
  int join_warps;   // of a row in the joining kernel
  int box;          // positions of a TMA box: a page, or an even part of it; 0: none, rows are gathered
  int keys_max;     // positions that the table can hold
  int prefix;       // min(shared_len, keys_max)
  float scale_log2;
  bool q_wide, o_wide;  // q rows can be read, rows of out written, four bytes at a time
  int4* rows;       // for the joining kernel: each token's Row,
  int2* seg_parts;  // the first and the last part of each segment,
  int2* seg_ctas;   // and the first and last CTA of each segment of the prefix's own tiles
  float* part;      // slots of kRows (m, l) and o
  int dim_padded;
  // The prefix on the tensor cores' own tiles (attention_tile.cuh), where on_tiles is set:
  bool on_tiles, q_copies;           // q_copies: q rows can be copied 16 bytes at a time
  int tile_rt, tile_streams;         // blocks of kTileRows rows of a segment; softmax warpgroups of a CTA
  int tile_segs, tiles_each;         // segments of a kv head, steps (of tile_streams / tile_rt key tiles) of each
  int tiles_total;                   // steps in all
  Costs cost;
  float* tile_part;                  // slots of kTileRows (m, l) and o
};

// What the joining kernel has to know of a token, as an int4: x its sequence's first segment (-1: no keys of
// its own), y its first row among the sequence's rows, z the first segment of the prefix (-1: it does not see
// it, or there is none; 0 where the prefix has its own tiles), w whether any sequence owns it.

// The cut of the work: prefix sums over the sequences (index B: the shared prefix). Tiles before, and
// segments before, each sequence; its first query row; its length.
struct Plan {
  int *tiles, *segs, *q0, *len;  // [B + 2], [B + 2], [B + 1], [B + 1] (len[B]: of the prefix, 0 if nobody sees it)
};
__host__ __device__ inline int plan_ints(int B) { return 4 * (B + 2) + 4; }

__host__ __device__ __forceinline__ Plan plan_of(int* base, int B) {
  return Plan{base + 4, base + 4 + (B + 2), base + 4 + 2 * (B + 2), base + 4 + 3 * (B + 2)};
}

__host__ __device__ __forceinline__ int seq_rows(const Plan& pl, int b) { return pl.q0[b + 1] - pl.q0[b]; }

// Whether every row of a sequence sees the whole prefix. The rows of one that does not (it ends inside
// the prefix, or is empty) take no part in the prefix's segments: it has all its keys for its own, so
// that those segments need no mask for rows, and what they hold cannot reach a row that must not see it.
__host__ __device__ __forceinline__ bool sees_prefix(const AttnParams& p, const Plan& pl, int b) {
  const int n = seq_rows(pl, b);
  return n > 0 && pl.len[b] - n + 1 >= p.prefix;
}

// The list's entry b: its query rows, and the keys of its tiles.
struct Entry {
  int rows, keys;
};
__host__ __device__ __forceinline__ Entry entry_of(const AttnParams& p, const Plan& pl, int b, int B) {
  Entry e;
  if (b < B) {
    e.rows = seq_rows(pl, b) * p.group;
    e.keys = min(pl.len[b], p.keys_max);
    if (sees_prefix(p, pl, b)) e.keys = e.keys > p.prefix ? e.keys - (p.prefix & -p.tile) : 0;
  } else {
    e.rows = p.on_tiles ? 0 : (int)p.a.tokens * p.group;  // the prefix has a list of its own then
    e.keys = pl.len[B];
  }
  return e;
}
__host__ __device__ __forceinline__ int blocks_of(const Entry& e) { return (e.rows + kRows - 1) / kRows; }
__host__ __device__ __forceinline__ int tiles_of(const AttnParams& p, const Entry& e) { return (e.keys + p.tile - 1) >> p.tile_shift; }

// Built by all threads of a CTA in its shared memory; base[0] = the parts' tiles in all, base[1] = parts in
// use, base[2] = CTAs that work on the prefix's own tiles (the first ones), by the two sides' cost.
__device__ void build_plan(const AttnParams& p, int* base) {
  const int B = (int)p.a.kv.seqs, T = (int)p.a.tokens, H = (int)p.a.kv.kv_heads;
  const Plan pl = plan_of(base, B);
  __shared__ int s_any, s_bad, s_warp_t[32], s_warp_s[32];
  __shared__ unsigned long long s_best;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_any = s_bad = 0, s_best = ~0ull;
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
  }
  __syncthreads();  // len[B], and the starts
  // Inclusive sums over runs of consecutive sequences, one run a thread.
  const int n = B + 1, per = (n + (int)blockDim.x - 1) / (int)blockDim.x, b0 = min(tid * per, n), b1 = min(b0 + per, n);
  int st = 0, ss = 0;
  for (int pass = 0; pass < 2; pass++) {
    for (int b = b0; b < b1; b++) {
      const Entry e = entry_of(p, pl, b, B);
      const int segs = blocks_of(e) * H;
      if (pass) pl.tiles[b] = st, pl.segs[b] = ss;
      st += segs * tiles_of(p, e);
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
  // CTAs for the prefix: as many as end soonest. The worst of them begins as many segments as its share can touch,
  // one where the CTAs are a multiple of the segments; the others are bound by HBM where there are many.
  const int steps = p.on_tiles && pl.len[B] ? p.tiles_total : 0, tiles = pl.tiles[n];
  if (steps) {
    const int segments = H * p.tile_segs;
    unsigned long long best = ~0ull;
    for (int x = tid + 1; x <= min(p.ctas, steps); x += blockDim.x) {
      if (x == p.ctas && tiles) break;
      const int share = (steps + x - 1) / x;
      const int touched = x % segments == 0 ? 1 : segments % x == 0 ? segments / x : (share - 2) / p.tiles_each + 2;
      const int64_t mine = (int64_t)share * p.cost.step + (int64_t)touched * p.cost.tile_segment;
      int64_t others = 0;
      if (tiles)
        others = max(((int64_t)tiles * p.cost.tile + (int64_t)pl.segs[n] * p.cost.segment) / (p.ctas - x), (int64_t)tiles * p.cost.tile_bytes / kBytesPerCycle) + p.cost.begin;
      best = min(best, (unsigned long long)max(mine, others) << 16 | (unsigned)x);
    }
    if (best != ~0ull) atomicMin(&s_best, best);
  }
  __syncthreads();
  if (tid == 0) {
    const int x = steps ? (int)(s_best & 0xffffu) : 0;
    base[0] = tiles;
    base[1] = (int)min((int64_t)tiles, (int64_t)(p.ctas - x) * p.warps);
    base[2] = x;
    base[3] = pl.segs[B];
  }
  __syncthreads();
}

// Part w of W covers tiles [first(w), first(w + 1)) of `total`.
__host__ __device__ __forceinline__ int first_tile(int total, int W, int w) { return (int)((int64_t)total * w / W); }

// Where a part stands: sequence, row block, head, tile. Tiles lie on multiples of their size, so that pages
// and boxes do not straddle them: the first one of a sequence behind the prefix may begin inside it.
struct __align__(16) Cursor {
  int b, mb, g, t, nt;  // nt tiles in a segment of b
  int mbs;              // row blocks of b
  int lo, end;          // of b: its keys; the first tile lies at lo, rounded down
};

__host__ __device__ __forceinline__ void enter(const AttnParams& p, const Plan& pl, int B, Cursor& c) {
  const Entry e = entry_of(p, pl, c.b, B);
  c.mbs = blocks_of(e);
  c.nt = c.mbs ? tiles_of(p, e) : 0;
  c.lo = c.b < B && sees_prefix(p, pl, c.b) ? p.prefix : 0;
  c.end = c.b < B ? min(pl.len[c.b], p.keys_max) : pl.len[B];
}

__host__ __device__ __forceinline__ Cursor seek(const AttnParams& p, const Plan& pl, int B, int tile) {
  int lo = 0, hi = B;  // the last index whose tiles begin at or before `tile`
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (pl.tiles[m] <= tile) lo = m;
    else hi = m - 1;
  }
  Cursor c;
  c.b = lo;
  enter(p, pl, B, c);
  const int at = tile - pl.tiles[lo], seg = c.nt ? at / c.nt : 0, H = (int)p.a.kv.kv_heads;
  c.t = at - seg * c.nt;
  c.mb = seg / H;
  c.g = seg - c.mb * H;
  return c;
}

// The next tile; t = 0 where it begins another segment. Never called behind the last tile.
__host__ __device__ __forceinline__ void advance(const AttnParams& p, const Plan& pl, int B, Cursor& c) {
  if (++c.t < c.nt) return;
  c.t = 0;
  if (++c.g == (int)p.a.kv.kv_heads) {
    c.g = 0;
    if (++c.mb == c.mbs) {
      c.mb = 0;
      do {
        if (++c.b <= B) enter(p, pl, B, c);
      } while (c.b <= B && c.nt == 0);
    }
  }
}

// The first and last of a segment's parts, as the joining kernel finds them: whether they are parts of `most`. It
// follows no others.
__host__ __device__ inline bool parts_ok(int2 w, int most) { return w.x >= 0 && w.x <= w.y && w.y < most; }

// The sequence that owns a row of q, or -1.
__host__ __device__ __forceinline__ int owner(const Plan& pl, int B, int token) {
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
// The softmax weights' scale. They are rounded to the cache's type for the second product. bf16 has the range of 32
// bits, and each weight keeps its precision. f16 has not: below 2^-14 it holds multiples of 2^-24 only, and a thousand
// small weights beside a large one lose the sum that the division counts (20000 keys of e^-17 of the largest weight
// each came out 44 % too heavy). So they are taken 2^up larger: relative to a maximum that is lower by `up`. The
// parts' running maximum is exact, their largest weight 2^15 of f16's 2^16; the tiles' may be 2^grow old. Weights down
// to 2^-29 (2^-25 .. 2^-29 in the tiles) of the largest keep f16's precision, smaller ones are off by 2^-40 (2^-36) of it.
// What f16's weights are relative to is rounded up, so that none leaves the type however coarse 32 bits are there.
template <typename T>
struct Weights {
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr float up = kHalf ? 15.0f : 0.0f, tile_up = kHalf ? 11.0f : 0.0f, tile_grow = kHalf ? 4.0f : 8.0f;
  // Of the largest product `x`, what its weights are relative to.
  static __device__ __forceinline__ float base(float x, float scale, float lower) {
    return kHalf ? __fmaf_ru(x, scale, -lower) : x * scale;
  }
};
template <typename T>
__device__ __forceinline__ void store_pair(const AttnParams& p, T* out, float a, float b) {
  if (p.o_wide) {
    *reinterpret_cast<uint32_t*>(out) = pack2<T>(a, b);
  } else {
    out[0] = from_f32<T>(a);
    out[1] = from_f32<T>(b);
  }
}
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.0f ? -INFINITY : ((m == -INFINITY ? 0.0f : m) + log2f(l)) * 0.69314718055994531f;
}
// Whether either half of a word is an infinity or a NaN (an exponent of ones carries into the sign's place): not 0.
template <typename T>
__device__ __forceinline__ uint32_t odd_word(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t one = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  return ((w & e) + one) & 0x80008000u;
}

}  // namespace
}  // namespace vtq
