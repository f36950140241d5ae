// attention_paged.cu -- attention of a batch's newest tokens over a paged key / value cache, with a
// prefix that all sequences share.
//
//   out = softmax(scale q k^T) v, one pass over the keys with the running maximum m and sum l of each
//   row's softmax:  m' = max(m, max s),  l' = l 2^(m - m') + sum 2^(s - m'),  o' likewise,
// scores in units of log2. The keys of a sequence are cut where it suits the machine; each part leaves
// (m, l, o) and attention_join_kernel adds the parts of a row.
//
// Work is a list of segments: (sequence, block of 16 query rows, kv head) over the sequence's own keys. A
// row is one query head of one token: the heads of a kv head and the drafted tokens of a sequence fill the
// rows of the MMA. The list is cut into equal runs of key tiles, one run a warp, whatever the lengths are
// (attention_part.cuh). The shared prefix is one more entry of the list, with the rows of all sequences;
// where that would take longer (many rows, a long prefix), it is a list of its own, cut over CTAs with blocks
// of 128 rows on tcgen05 (attention_tile.cuh), and both run side by side: one is bound by HBM, the other by
// the tensor cores and the softmax, so the SMs are dealt between them by cost. Every CTA derives the same
// cut from the lengths on the device (attention_plan.cuh, 2 us); the host never needs them.
#include <algorithm>

#include "attention_part.cuh"
#include "attention_tile.cuh"

namespace vtq {

vtq_status serve_check_kv(const char* fn, const vtq_paged_kv& kv);

namespace {

// Shapes of the two roles by head_dim (rounded up to 64, 128, 256) and blocks of rows of the prefix.
template <typename T, int DP>
struct Part;
template <typename T>
struct Part<T, 64> { static constexpr int KT = 32, WARPS = 12; };
template <typename T>
struct Part<T, 128> { static constexpr int KT = 32, WARPS = 12; };
template <typename T>
struct Part<T, 256> { static constexpr int KT = 16, WARPS = 8; };
template <typename T, int DP, int RT>
struct Tile;
template <typename T, int RT>
struct Tile<T, 64, RT> { static constexpr int KT = 128, STREAMS = 2, NSLOT = 8; };
template <typename T, int RT>
struct Tile<T, 128, RT> { static constexpr int KT = 128, STREAMS = 2, NSLOT = RT == 2 ? 5 : 6; };
template <typename T>
struct Tile<T, 256, 1> { static constexpr int KT = 64, STREAMS = 1, NSLOT = 5; };

template <typename T, int DP, int RT>
constexpr int attention_threads() {
  if constexpr (RT == 0) return 32 * Part<T, DP>::WARPS;
  else return TileShape<T, DP, Tile<T, DP, RT>::KT, RT, Tile<T, DP, RT>::STREAMS, Tile<T, DP, RT>::NSLOT>::THREADS;
}

// RT = 0: no prefix of its own.
template <typename T, int DP, int RT>
__global__ void __launch_bounds__(attention_threads<T, DP, RT>(), 1)
    attention_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap tmk,
                     const __grid_constant__ CUtensorMap tmv) {
  using P = Part<T, DP>;
  using PS = PartShape<T, DP, P::KT, P::WARPS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  int* base = reinterpret_cast<int*>(smem + PS::STAGES_BYTES);
  tc5::grid_wait();
  tc5::grid_release();
  build_plan(p, base);
  const int cta = (int)blockIdx.x, x = base[2];
  if (cta == p.ctas - 1) {
    const int B = (int)p.a.kv.seqs;
    const Plan pl = plan_of(base, B);
    for (int i = threadIdx.x; i < (int)p.a.tokens; i += blockDim.x) {
      const int b = owner(pl, B, i);
      int4 r = make_int4(-1, 0, -1, b >= 0);
      if (b >= 0) {
        if (pl.tiles[b + 1] > pl.tiles[b]) r.x = pl.segs[b];
        r.y = (i - pl.q0[b]) * p.group;
        if (pl.len[B] && sees_prefix(p, pl, b)) r.z = p.on_tiles ? 0 : base[3];
      }
      p.rows[i] = r;
    }
    if (p.a.status)
      for (int b = threadIdx.x; b < B; b += blockDim.x)
        if (pl.len[b] > p.keys_max || p.a.kv_len[b] < 0) atomicOr(p.a.status, SERVE_BAD_INDEX);
  }
  if constexpr (RT > 0) {
    if (cta < x) {
      using S = Tile<T, DP, RT>;
      __syncthreads();  // the plan has been read: the ring takes its place
      tile_role<T, DP, S::KT, RT, S::STREAMS, S::NSLOT>(p, tmk, tmv, smem, cta, x);
      return;
    }
  }
  part_role<T, DP, P::KT, P::WARPS, RT == 0>(p, tmk, tmv, smem, base, cta - x, p.ctas - x);
}

// Adds the parts of each row (query head of a token): p.join_warps warps a row, one where the rows fill the SMs, more
// where they are few and their parts many (one sequence of 4096 keys, 32 rows: 38 us with one). A row whose keys one part took alone is
// there already. The kernel before lets this one start early; until it is done the warps of the first wave go
// through their own code once, on made-up places and with nothing stored, so that the instructions are there
// when the parts are (8 us for 128 rows without). What is left is a chain of four reads from L2: a row's entry, its
// parts' numbers, their (m, l) and first values at once, and their further values.
constexpr int kJoinWarps = 8;  // of a block
template <typename T, int DP>
__global__ void __launch_bounds__(32 * kJoinWarps, DP > 128 ? 2 : 3) attention_join_kernel(const __grid_constant__ AttnParams p) {
  const int lane = threadIdx.x & 31;
  __shared__ float s_acc[kJoinWarps][DP];
  const int warp = threadIdx.x >> 5, split = p.join_warps, sub = warp % split;
  const int row = ((int)blockIdx.x * kJoinWarps + warp) / split;
  const int heads = (int)p.a.heads, H = (int)p.a.kv.kv_heads, D = (int)p.a.kv.head_dim;
  if (row >= (int)p.a.tokens * heads) return;
  const int token = row / heads, head = row - token * heads, g = head / p.group;
#pragma unroll 1
  for (int pass = (int)blockIdx.x < 4 * p.ctas ? 0 : 1; pass < 2; pass++) {
    if (pass) tc5::grid_wait();
    int4 of = make_int4(0, 0, p.prefix ? 0 : -1, 1);
    if (pass) of = p.rows[token];
    if (!of.w) {  // no sequence owns the row
      if ((p.a.clear & 1u) && !sub)
        for (int d = lane; d < D; d += 32) static_cast<T*>(p.a.out)[token * p.a.o_tok + head * p.a.o_head + d] = from_f32<T>(0.0f);
      if ((p.a.clear & 2u) && p.a.lse && !sub && !lane) p.a.lse[token * p.a.lse_tok + head] = -INFINITY;
      return;
    }
    // The parts of the row's place among the sequence's own rows, and among all rows for the prefix.
    int count[2] = {0, 0}, rr[2] = {0, 0};
    const float* slot0[2] = {p.part, p.part};
    bool lost = false;
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int seg0 = k ? of.z : of.x;
      if (seg0 < 0) continue;
      const int r = (k ? token * p.group : of.y) + head - g * p.group;
      const bool tiles = k && p.on_tiles;
      // A CTA of the prefix's own tiles leaves a part for each stream: of other rows, or of the same rows'
      // other keys.
      const int seg = tiles ? g * p.tile_segs + r / (kTileRows * p.tile_rt) : seg0 + r / kRows * H + g;
      int2 w = make_int2(0, 0);
      if (pass) {
        w = (tiles ? p.seg_ctas : p.seg_parts)[seg];
        // What the kernel before left for every segment, also where a wait of its ran out; nothing else is followed.
        if (!parts_ok(w, tiles ? min(p.ctas, p.tiles_total) : p.ctas * p.warps)) {
          if (p.a.status) atomicOr(p.a.status, KERR_TIMEOUT);
          lost = true;
          continue;
        }
      }
      rr[k] = r % (tiles ? kTileRows : kRows);
      count[k] = (w.y - w.x + 1) * (tiles && p.tile_rt == 1 ? p.tile_streams : 1);
      if (!pass) continue;
      slot0[k] = tiles ? p.tile_part + ((int64_t)(w.x + seg) * p.tile_streams + (p.tile_rt == 2 ? r / kTileRows % 2 : 0)) * (kTileRows * (DP + 2))
                       : p.part + (int64_t)(w.x + seg) * (kRows * (DP + 2));
    }
    if (!pass) rr[0] = rr[1] = 0;
    const int parts = count[0] + count[1];
    if (pass && !p.on_tiles && count[0] == 1 && of.z < 0) return;  // written by the part
    // Part i's (m, l) of the row, and its o.
    auto at = [&](int i, const float*& o) {
      const bool k = i >= count[0], tiles = k && p.on_tiles;
      const int rows = tiles ? kTileRows : kRows, step = rows * (DP + 2) * (tiles && p.tile_rt == 2 ? 2 : 1);
      const float* s = (k ? slot0[1] : slot0[0]) + (pass ? (int64_t)(i - (k ? count[0] : 0)) * step : 0);
      const int r = k ? rr[1] : rr[0];
      o = s + (pass ? 2 * rows : 0) + r * DP;
      return s + 2 * r;
    };
    constexpr int kAtOnce = DP > 128 ? 4 : 8, V = DP / 32;  // parts read together; values a lane
    float v[kAtOnce][V];
    // Each lane finds one part's place, which all load from together.
    const float* place;
    auto find = [&](int i) { return *reinterpret_cast<const float2*>(at(max(min(i, parts - 1), 0), place)); };
    auto load = [&](int i) {
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const float* s = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(place), (i + k) & 31));
        if constexpr (V == 2) {
          const float2 x = *reinterpret_cast<const float2*>(s + 2 * lane);
          v[k][0] = x.x, v[k][1] = x.y;
        } else {
#pragma unroll
          for (int e = 0; e < V; e += 4) {
            const float4 x = *reinterpret_cast<const float4*>(s + 32 * e + 4 * lane);
            v[k][e] = x.x, v[k][e + 1] = x.y, v[k][e + 2] = x.z, v[k][e + 3] = x.w;
          }
        }
      }
    };
    // This warp's parts, and all parts' (m, l).
    const int lo = parts * sub / split, hi = parts * (sub + 1) / split;
    const float* unused;
    const float2 none = make_float2(-INFINITY, 0.0f);
    constexpr int kMl = 4;
    float2 ml[kMl];
#pragma unroll
    for (int j = 0; j < kMl; j++)
      ml[j] = lane + 32 * j < parts ? *reinterpret_cast<const float2*>(at(lane + 32 * j, unused)) : none;
    float2 mine = find(lo + lane);
    load(0);
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kMl; j++) m = fmaxf(m, ml[j].x);
#pragma unroll 1
    for (int i = lane + 32 * kMl; i < parts; i += 32) m = fmaxf(m, *at(i, unused));
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float um = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, f = 0.0f, acc[V];
#pragma unroll
    for (int j = 0; j < kMl; j++) l += exp2_fast(ml[j].x - um) * ml[j].y;
#pragma unroll 1
    for (int i = lane + 32 * kMl; i < parts; i += 32) {
      const float2 x = *reinterpret_cast<const float2*>(at(i, unused));
      l += exp2_fast(x.x - um) * x.y;
    }
#pragma unroll
    for (int e = 0; e < V; e++) acc[e] = 0.0f;
#pragma unroll 1
    for (int i = lo; i < hi; i += kAtOnce) {
      if ((i - lo) % 32 == 0) {
        if (i > lo) mine = find(i + lane);
        f = mine.y == 0.0f ? 0.0f : exp2_fast(mine.x - um);  // nothing in it, whatever its o holds
      }
      if (i > lo) load(i - lo);
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const float fk = __shfl_sync(0xffffffffu, f, (i - lo + k) & 31);
#pragma unroll
        for (int e = 0; e < V; e++)
          if (i + k < hi && fk != 0.0f) acc[e] = fmaf(fk, v[k][e], acc[e]);
      }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    if (split > 1) {
      // The row's warps add theirs in order; a barrier of their own, as other rows of the block may have left.
#pragma unroll
      for (int e = 0; e < V; e++) s_acc[warp][e * 32 + lane] = acc[e];
      asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / split), "r"(32 * split) : "memory");
      if (sub == 0)
        for (int w = 1; w < split; w++)
#pragma unroll
          for (int e = 0; e < V; e++) acc[e] += s_acc[warp + w][e * 32 + lane];
      asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / split), "r"(32 * split) : "memory");
      if (sub) continue;
    }
    if (lost) l = __uint_as_float(0x7fc00000u);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key: zeros
    T* out = static_cast<T*>(p.a.out) + token * p.a.o_tok + head * p.a.o_head;
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const int d = V == 2 ? 2 * lane : 32 * (e & ~3) + 4 * lane + (e & 2);
      if (pass && d < D) store_pair<T>(p, out + d, acc[e] * inv, acc[e + 1] * inv);
    }
    if (pass && p.a.lse && lane == 0) p.a.lse[token * p.a.lse_tok + head] = lse_of(m, l);
  }
}

int padded_dim(int64_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
int part_warps(int dp) { return dp == 64 ? Part<__half, 64>::WARPS : dp == 128 ? Part<__half, 128>::WARPS : Part<__half, 256>::WARPS; }

// Fitted to when the two kinds of CTA end, on batches of 16 .. 256 sequences behind 8199 .. 32768 keys. A step is 128
// keys and 256 rows, 64 keys and 128 rows at head_dim 256; a part's tile 32 keys, 16 there.
Costs costs(int dp) {
  Costs c;
  c.tile = dp == 64 ? 315 : dp == 128 ? 540 : 660;
  c.segment = 300;
  c.begin = 25000;  // until the last of the parts is done: a warp by itself is slow
  c.step = dp == 64 ? 4000 : dp == 128 ? 4900 : 3050;
  c.tile_segment = 10000;
  c.tile_bytes = (dp == 256 ? 16 : 32) * dp * 4;
  return c;
}

// How the prefix goes to the tensor cores' own tiles, and where: more rows than the 16 that one read of
// a key serves in the part kernel, and work enough that they end sooner than parts would, by the same costs
// (parts and tiles, 8 kv heads of 4 rows a token: 64 tokens behind 500 keys 22 and 26 us, 30 behind 1000 23 and
// 23, behind 2000 28 and 29, 64 behind 1000 29 and 26, behind 2000 40 and 27, 40 behind 6000 53 and 27).
struct TileCut {
  bool on;
  int keys, rt, streams, segs, each;  // keys of a tile; see AttnParams
  int64_t total;
};
TileCut tile_cut(const vtq_attention_args& a) {
  TileCut c = {};
  const int64_t rows = a.tokens * (a.heads / a.kv.kv_heads), prefix = std::min(a.shared_len, a.kv.table_width * a.kv.page_size);
  const bool wide = a.kv.head_dim > 128;
  c.keys = wide ? 64 : 128;
  c.streams = wide ? 1 : 2;
  c.rt = !wide && rows > kTileRows ? 2 : 1;
  c.segs = (int)((rows + kTileRows * c.rt - 1) / (kTileRows * c.rt));
  const int step = c.keys * c.streams / c.rt;
  c.each = (int)((prefix + step - 1) / step);
  c.total = a.kv.kv_heads * (int64_t)c.segs * c.each;
  if (rows <= kRows || !prefix) return c;
  const Costs cost = costs(padded_dim(a.kv.head_dim));
  const int64_t sms = num_sms(), share = (c.total + sms - 1) / sms, key_tiles = (prefix + (wide ? 15 : 31)) / (wide ? 16 : 32);
  const int64_t parts = (rows + kRows - 1) / kRows * a.kv.kv_heads * key_tiles * cost.tile / sms + cost.begin / 5;
  c.on = share * cost.step + ((share + c.each - 1) / c.each) * cost.tile_segment < parts;
  return c;
}
size_t tile_bytes(const vtq_attention_args& a) {
  const TileCut c = tile_cut(a);
  if (!c.on) return 0;
  const int64_t slots = (std::min<int64_t>(c.total, num_sms()) + a.kv.kv_heads * c.segs) * c.streams;
  return (size_t)slots * kTileRows * (padded_dim(a.kv.head_dim) + 2) * 4;
}

// Segments of any lengths: each sequence's rows and, once more, all rows for the prefix.
int64_t most_segments(const vtq_attention_args& a) {
  const int64_t group = a.heads / a.kv.kv_heads, rows = a.tokens * group;
  return (rows / kRows + a.kv.seqs + (a.shared_len && !tile_cut(a).on ? (rows + kRows - 1) / kRows : 0)) * a.kv.kv_heads;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
size_t row_bytes(const vtq_attention_args& a) { return up256((size_t)a.tokens * sizeof(int4)); }
size_t seg_bytes(const vtq_attention_args& a) { return up256((size_t)most_segments(a) * sizeof(int2)); }
size_t cta_bytes(const vtq_attention_args& a) {
  const TileCut c = tile_cut(a);
  return c.on ? up256((size_t)a.kv.kv_heads * c.segs * sizeof(int2)) : 0;
}
size_t part_bytes(const vtq_attention_args& a) {
  const int dp = padded_dim(a.kv.head_dim);
  const int64_t slots = most_segments(a) + (int64_t)num_sms() * part_warps(dp);
  return up256((size_t)slots * kRows * (dp + 2) * 4);
}

vtq_status check(const char* fn, const vtq_attention_args* a) {
  if (!a) return serve_fail(VTQ_ERR_INVALID_ARG, "%s: null arguments", fn);
  if (vtq_status s = serve_check_kv(fn, a->kv)) return s;
  if (a->tokens < 0 || a->heads < 1 || a->heads % a->kv.kv_heads || a->shared_len < 0)
    return serve_fail(VTQ_ERR_INTERNAL, "%s: bad shape (heads not a multiple of kv_heads, or a negative size)", fn);
  if (a->kv.seqs > kMaxSeqs)
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (over %d sequences in one call)", fn, kMaxSeqs);
  if (a->tokens > (1 << 20) || a->heads > 65536 || a->tokens * a->heads > INT32_MAX / 2 || a->kv.table_width > INT32_MAX / 2 / a->kv.page_size)
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (over 2^20 tokens, 2^16 heads or 2^30 positions)", fn);
  const int64_t tiles = (a->kv.table_width * a->kv.page_size + 15) / 16 + 1;
  if (most_segments(*a) * tiles > INT32_MAX || tile_cut(*a).total > INT32_MAX)
    return serve_fail(VTQ_ERR_NOT_IMPLEMENTED, "%s: not implemented (query rows times table positions over 2^35)", fn);
  return VTQ_OK;
}

template <typename T, int DP, int RT>
cudaError_t launch(AttnParams p, cudaStream_t st) {
  using P = Part<T, DP>;
  size_t smem = PartShape<T, DP, P::KT, P::WARPS>::smem((int)p.a.kv.seqs);
  if constexpr (RT > 0) {
    using S = Tile<T, DP, RT>;
    smem = std::max(smem, TileShape<T, DP, S::KT, RT, S::STREAMS, S::NSLOT>::SMEM);
  }
  smem += 1024;  // alignment
  p.warps = P::WARPS;
  p.tile = P::KT;
  p.tile_shift = P::KT == 32 ? 5 : 4;
  auto kernel = attention_kernel<T, DP, RT>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem((const void*)kernel, smem, allowed);
  if (e != cudaSuccess) return e;
  // A box is the largest power of two of positions that pages are made of.
  CUtensorMap tmk = {}, tmv = {};
  const vtq_paged_kv& kv = p.a.kv;
  p.box = 1;
  while (p.box < P::KT && kv.page_size % (2 * p.box) == 0) p.box *= 2;
  if (p.box < 4) {
    p.box = 0;
  } else {
    const uint64_t dim[4] = {(uint64_t)kv.head_dim, (uint64_t)kv.page_size, (uint64_t)kv.kv_heads, (uint64_t)kv.pages};
    const uint64_t ks[3] = {2 * (uint64_t)kv.k_slot, 2 * (uint64_t)kv.k_head, 2 * (uint64_t)kv.k_page};
    const uint64_t vs[3] = {2 * (uint64_t)kv.v_slot, 2 * (uint64_t)kv.v_head, 2 * (uint64_t)kv.v_page};
    if (tma_half_map(&tmk, kv.k, dim, ks, 64, (uint32_t)p.box) != cudaSuccess ||
        tma_half_map(&tmv, kv.v, dim, vs, 64, (uint32_t)p.box) != cudaSuccess)
      p.box = 0;  // strides that TMA does not take: rows are gathered
  }
  e = launch_after(kernel, dim3((unsigned)p.ctas), attention_threads<T, DP, RT>(), smem, 1, st, p, tmk, tmv);
  if (e != cudaSuccess) return e;
  const int64_t rows = p.a.tokens * p.a.heads;
  p.join_warps = 1;
  while (p.join_warps < kJoinWarps && rows * p.join_warps * 2 <= 16 * p.ctas) p.join_warps *= 2;
  const int64_t blocks = (rows * p.join_warps + kJoinWarps - 1) / kJoinWarps;
  return launch_after(attention_join_kernel<T, DP>, dim3((unsigned)blocks), 32 * kJoinWarps, 0, 1, st, p);
}

template <typename T>
cudaError_t launch_dim(const AttnParams& p, cudaStream_t st) {
  const int rt = p.on_tiles ? p.tile_rt : 0;
  switch (p.dim_padded) {
    case 64: return rt == 2 ? launch<T, 64, 2>(p, st) : rt ? launch<T, 64, 1>(p, st) : launch<T, 64, 0>(p, st);
    case 128: return rt == 2 ? launch<T, 128, 2>(p, st) : rt ? launch<T, 128, 1>(p, st) : launch<T, 128, 0>(p, st);
    default: return rt ? launch<T, 256, 1>(p, st) : launch<T, 256, 0>(p, st);
  }
}

}  // namespace
}  // namespace vtq

using namespace vtq;

extern "C" {

size_t vtq_attention_paged_workspace_bytes(const vtq_attention_args* a) {
  if (check("vtq_attention_paged", a) || a->tokens == 0 || a->kv.seqs == 0) return 0;
  return row_bytes(*a) + seg_bytes(*a) + cta_bytes(*a) + part_bytes(*a) + tile_bytes(*a);
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
  p.by_group = divisor(p.group);
  p.by_page = divisor(a->kv.page_size);
  p.dim_padded = padded_dim(a->kv.head_dim);
  p.ctas = num_sms();
  p.keys_max = (int)(a->kv.table_width * a->kv.page_size);
  p.prefix = (int)std::min<int64_t>(a->shared_len, p.keys_max);
  // A scale of 0 weighs every key alike; so does the smallest number, with which no finite score is above 2^-20 (and
  // which leaves the -inf of masked keys what it is).
  p.scale_log2 = a->scale == 0.0f ? 1.4e-45f : a->scale * 1.4426950408889634f;
  p.q_wide = (reinterpret_cast<uintptr_t>(a->q) & 3u) == 0 && a->q_tok % 2 == 0 && a->q_head % 2 == 0;
  p.o_wide = (reinterpret_cast<uintptr_t>(a->out) & 3u) == 0 && a->o_tok % 2 == 0 && a->o_head % 2 == 0;
  uint8_t* at = static_cast<uint8_t*>(ws);
  p.rows = reinterpret_cast<int4*>(at);
  p.seg_parts = reinterpret_cast<int2*>(at += row_bytes(*a));
  p.seg_ctas = reinterpret_cast<int2*>(at += seg_bytes(*a));
  p.part = reinterpret_cast<float*>(at += cta_bytes(*a));
  const TileCut c = tile_cut(*a);
  p.on_tiles = c.on;
  if (c.on) {
    p.q_copies = aligned16(a->q) && a->q_tok % 8 == 0 && a->q_head % 8 == 0;
    p.tile_rt = c.rt;
    p.tile_streams = c.streams;
    p.tile_segs = c.segs;
    p.tiles_each = c.each;
    p.tiles_total = (int)c.total;
    p.cost = costs(p.dim_padded);
    p.tile_part = reinterpret_cast<float*>(at + part_bytes(*a));
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return serve_cuda(a->kv.dtype == VTQ_F16 ? launch_dim<__half>(p, st) : launch_dim<__nv_bfloat16>(p, st), fn);
}

}  // extern "C"
