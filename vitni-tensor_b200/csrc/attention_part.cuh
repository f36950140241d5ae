// attention_part.cuh -- attention_paged: the sequences' own keys, and a prefix too short or for too few rows
// to pay for attention_tile.cuh.
//
// A warp takes a run of key tiles by itself: 16 query rows against KT keys a step with mma.sync (4 of the 16
// rows are real where a kv head has 4 query heads and a sequence one token: what counts is that the keys
// arrive) and no barrier but its own. Bound: HBM by bytes, and close behind it the latency of a warp's own
// instructions (5100 cycles a tile, 2000 of them the scores), so that warps count more than tiles in flight:
// 12 of them with one K and one V tile each, the next K asked for behind this one's scores, the next V behind
// this one's sum, the next segment's queries behind its last weights. A new segment costs a warp 3000 cycles
// beside its tiles. Tiles come by TMA, a box for each page or even piece of one, where pages hold 4 positions
// or more.
#pragma once
#include "attention_plan.cuh"

namespace vtq {
namespace {

// DP: head_dim rounded up to what the MMA loop takes (64, 128, 256).
template <typename T, int DP, int KT, int WARPS>
struct PartShape {
  static constexpr uint32_t TILE = KT * DP * 2, STAGES_BYTES = WARPS * 2 * TILE;
  static constexpr size_t smem(int B) { return STAGES_BYTES + (plan_ints(B) * 4 + 15) / 16 * 16 + (size_t)WARPS * KT * sizeof(longlong2); }
};

// The role of CTA `cta` of `ctas`; ALONE: none works on the prefix's own tiles; `base` is the plan, at smem + STAGES_BYTES.
template <typename T, int DP, int KT, int WARPS, bool ALONE>
__device__ __forceinline__ void part_role(const AttnParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv, uint8_t* smem,
                                          int* base, int cta, int ctas) {
  using L = PartShape<T, DP, KT, WARPS>;
  constexpr int CH = DP / 8;  // 16-byte chunks of a row
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int B = (int)p.a.kv.seqs, H = (int)p.a.kv.kv_heads, D = (int)p.a.kv.head_dim, page_size = (int)p.a.kv.page_size;
  __shared__ __align__(8) uint64_t s_full[WARPS][2];  // of the K tile, of the V tile
  // Where this tile and the next one stand, by turns: in shared memory, for the registers are all in use (a spill
  // costs the loop a quarter of its rate).
  __shared__ Cursor s_at[WARPS][2];
  if (warp >= WARPS) return;
  longlong2* rows = reinterpret_cast<longlong2*>(reinterpret_cast<uint8_t*>(base) + (plan_ints(B) * 4 + 15) / 16 * 16) + warp * KT;
  const Plan pl = plan_of(base, B);
  const int total = base[0], W = base[1];
  const int w = warp * ctas + cta;  // few parts spread over the SMs first
  if (w >= W) return;
  if (lane == 0) {
    for (int s = 0; s < 2; s++) tc5::bar_init(smem_u32(&s_full[warp][s]), 1);
    fence_mbar_init();
  }
  __syncwarp();
  const int tile0 = first_tile(total, W, w), tile1 = first_tile(total, W, w + 1);
  const uint32_t k_s = smem_u32(smem) + warp * 2 * L::TILE, v_s = k_s + L::TILE;
  const uint32_t k_full = smem_u32(&s_full[warp][0]), v_full = smem_u32(&s_full[warp][1]);
  // Blocks of 64 values, rows of 128 bytes, chunks swizzled as TMA does.
  auto swizzled = [](int key, int chunk) {
    return (uint32_t)((chunk >> 3) * (KT * 128) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4));
  };
  const int box = p.box < KT ? p.box : KT, boxes = box ? KT / box : 0, my_box = box ? lane / box : 0;

  // The row of the page table that a position of a sequence is read through.
  auto row_of = [&](const Cursor& c, int pos) { return c.b == B || (c.lo == 0 && pos < p.prefix) ? 0 : c.b; };
  // The page of this lane's box of a tile, asked for a tile ahead (-1 where the box has no key), and where in it.
  auto ask = [&](const Cursor& c) {
    const int pos = (c.lo & -KT) + c.t * KT + lane * box, at = p.by_page(pos);
    const bool in = lane < boxes && pos + box > c.lo && pos < c.end;
    return make_int2(in ? p.a.kv.table[row_of(c, pos) * p.a.kv.table_ld + at] : -1, pos - at * page_size);
  };
  // How the tile at a cursor comes: in boxes or, where there are none or one would straddle the end of the
  // prefix in a sequence that reads both sides of it, row by row.
  struct Tile {
    uint32_t valid, there;  // the keys, and the boxes, that are there
    int page, slot;         // of this lane's box
    bool by_box;
  };
  auto find = [&](const Cursor& c, int2 page) {
    Tile x;
    const int key0 = (c.lo & -KT) + c.t * KT;
    x.page = page.x;
    x.slot = page.y;
    x.there = 0;
    x.by_box = boxes && !(c.b < B && c.lo == 0 && key0 < p.prefix && key0 + KT > p.prefix && p.prefix % box);
    if (x.by_box) {
      const int pos = key0 + lane * box;
      const bool in = lane < boxes && pos + box > c.lo && pos < c.end, ok = in && page.x >= 0 && page.x < p.a.kv.pages;
      if (in && !ok && p.a.status) atomicOr(p.a.status, SERVE_BAD_INDEX);
      x.there = __ballot_sync(0xffffffffu, ok);
      x.valid = __ballot_sync(0xffffffffu, lane < KT && key0 + lane >= c.lo && key0 + lane < c.end && ((x.there >> my_box) & 1));
      return x;
    }
    bool ok = false;
    if (lane < KT) {
      const int pos = key0 + lane;
      int64_t ko = 0, vo = 0;
      if (pos >= c.lo && pos < c.end) {
        const int at = p.by_page(pos);
        const int64_t pg = p.a.kv.table[row_of(c, pos) * p.a.kv.table_ld + at], slot = pos - at * page_size;
        ok = pg >= 0 && pg < p.a.kv.pages;
        if (ok) {
          ko = pg * p.a.kv.k_page + slot * p.a.kv.k_slot + c.g * p.a.kv.k_head;
          vo = pg * p.a.kv.v_page + slot * p.a.kv.v_slot + c.g * p.a.kv.v_head;
        } else if (p.a.status) {
          atomicOr(p.a.status, SERVE_BAD_INDEX);
        }
      }
      rows[lane] = make_longlong2(ko, vo);
    }
    x.valid = __ballot_sync(0xffffffffu, ok);
    __syncwarp();
    return x;
  };
  // Starts the K (or V) tile of `x`, which stands at `c`. One copy group a call, whichever way: they are waited for by count.
  auto load = [&](const Tile& x, const Cursor& c, bool is_v) {
    const uint32_t dst = is_v ? v_s : k_s, full = is_v ? v_full : k_full;
    if (x.by_box) {
      if (lane == 0) tc5::bar_expect(full, __popc(x.there) * box * 128 * (DP / 64));
      __syncwarp();
      if ((x.there >> lane) & 1) {
#pragma unroll
        for (int h = 0; h < DP / 64; h++)
          tc5::tma_4d(dst + h * KT * 128 + lane * box * 128, is_v ? &tmv : &tmk, 64 * h, x.slot, c.g, x.page, full);
      }
    } else {
      const T* from = static_cast<const T*>(is_v ? p.a.kv.v : p.a.kv.k);
#pragma unroll 1
      for (int i = 0; i < KT * CH / 32; i++) {
        const int e = i * 32 + lane, key = e / CH, chunk = e - key * CH;
        const longlong2 o = rows[key];
        const bool there = ((x.valid >> key) & 1) && chunk * 8 < D;
        copy16(dst + swizzled(key, chunk), from + (there ? (is_v ? o.y : o.x) + chunk * 8 : 0), there);
      }
      if (lane == 0) tc5::bar_arrive(full);  // the tile's phase
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // The K (or V) tile of this step has landed. One group may still be out: the one started behind it.
  auto landed = [&](uint32_t full, uint32_t parity) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    const bool ok = tc5::bar_wait(full, parity);
    if (!ok && lane == 0 && p.a.status) atomicOr(p.a.status, KERR_TIMEOUT);
    __syncwarp();
    return ok;
  };

  Cursor* const at = s_at[warp];
  // Lane 0 writes the cursor behind `from` to `to`.
  auto step = [&](int from, int to) {
    if (lane == 0) {
      Cursor n = at[from];
      advance(p, pl, B, n);
      at[to] = n;
    }
    __syncwarp();
  };
  if (lane == 0) at[0] = seek(p, pl, B, tile0);
  __syncwarp();
  Tile next = find(at[0], ask(at[0]));
  load(next, at[0], false);
  load(next, at[0], true);
  int2 page = make_int2(-1, 0);
  if (tile0 + 1 < tile1) {
    step(0, 1);
    page = ask(at[1]);
  }

  uint32_t qf[DP / 16][4];
  float o[DP / 8][4];
  float m0 = 0, m1 = 0, l0 = 0, l1 = 0;
  int lim[2], lim_min, rows_in;         // how far the two rows of this lane see, and the least of all; rows there are
  // A negative scale is a positive one on queries of the other sign.
  const float scale = fabsf(p.scale_log2);
  const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
  const int r0 = lane >> 2, cq = 2 * (lane & 3);
  // A segment's 16 query rows. Those of the next one are asked for when the last scores of this one are there.
  auto queries = [&](const Cursor& c) {
    const bool shared = c.b == B;
    const int all = (shared ? (int)p.a.tokens : seq_rows(pl, c.b)) * p.group, q0 = shared ? 0 : pl.q0[c.b];
    const T* qr[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int row = c.mb * kRows + r0 + 8 * h, tok = p.by_group(row);
      qr[h] = row < all ? static_cast<const T*>(p.a.q) + (int64_t)(q0 + tok) * p.a.q_tok + (int64_t)(c.g * p.group + row - tok * p.group) * p.a.q_head : nullptr;
    }
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
  };
  queries(at[0]);
  // A wait that ran out ends the loads, and what this part has not left yet becomes NaN (its sums of weights are): the
  // joining kernel still finds an entry and a slot for each segment, and rows that lack keys show it. Copies on their
  // way then were asked for before that wait, 2 s ago.
  bool ok = true;
  for (int tile = tile0; tile < tile1; tile++) {
    const int turn = (tile - tile0) & 1;
    const Cursor& c = at[turn];
    if (tile == tile0 || c.t == 0) {
      const bool shared = c.b == B;
      const int n = shared ? (int)p.a.tokens : seq_rows(pl, c.b);
      rows_in = min(kRows, n * p.group - c.mb * kRows);
#pragma unroll
      for (int h = 0; h < 2; h++)
        lim[h] = shared ? INT32_MAX : min(pl.len[c.b] - n + p.by_group(c.mb * kRows + r0 + 8 * h) + 1, p.keys_max);
      lim_min = __reduce_min_sync(0xffffffffu, min(r0 < rows_in ? lim[0] : INT32_MAX, r0 + 8 < rows_in ? lim[1] : INT32_MAX));
      if (flip) {
#pragma unroll
        for (int k = 0; k < DP / 16; k++)
#pragma unroll
          for (int e = 0; e < 4; e++) qf[k][e] ^= flip;
      }
#pragma unroll
      for (int i = 0; i < DP / 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[i][e] = 0.0f;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.0f;
    }
    const uint32_t parity = (uint32_t)turn;
    const uint32_t valid = next.valid;
    ok = ok && landed(k_full, parity);
    const int key0 = (c.lo & -KT) + c.t * KT;
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
    __syncwarp();
    if (tile + 1 < tile1) {
      next = find(at[turn ^ 1], page);
      if (ok) load(next, at[turn ^ 1], false);
    } else {
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    float x0 = -INFINITY, x1 = -INFINITY;
    if (!whole) {
#pragma unroll
      for (int n = 0; n < KT / 8; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int j = 8 * n + cq + e;
          const bool there = (valid >> j) & 1;
          if (!there || key0 + j >= lim[0]) sc[n][e] = -INFINITY;
          if (!there || key0 + j >= lim[1]) sc[n][2 + e] = -INFINITY;
        }
    }
#pragma unroll
    for (int n = 0; n < KT / 8; n++) {
      x0 = fmaxf(fmaxf(sc[n][0], sc[n][1]), x0);
      x1 = fmaxf(fmaxf(sc[n][2], sc[n][3]), x1);
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
    }
    const float n0 = fmaxf(m0, Weights<T>::base(x0, scale, Weights<T>::up)), n1 = fmaxf(m1, Weights<T>::base(x1, scale, Weights<T>::up));
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
      const float e0 = exp2_fast(fmaf(sc[n][0], scale, -u0)), e1 = exp2_fast(fmaf(sc[n][1], scale, -u0));
      const float e2 = exp2_fast(fmaf(sc[n][2], scale, -u1)), e3 = exp2_fast(fmaf(sc[n][3], scale, -u1));
      l0 += e0 + e1;
      l1 += e2 + e3;
      // The weights are rounded to the cache's type for the second product: relative to each
      // weight (Weights), so a row's error stays that of its type, as the rounding of v itself.
      pf[n >> 1][2 * (n & 1)] = pack2<T>(e0, e1);
      pf[n >> 1][2 * (n & 1) + 1] = pack2<T>(e2, e3);
    }
    if (tile + 1 < tile1 && at[turn ^ 1].t == 0) queries(at[turn ^ 1]);
    ok = ok && landed(v_full, parity);
    if (!whole) {
      // A weight of 0 times an infinity or a NaN is no 0: keys that are not there (what lies behind a sequence's end
      // in its last page, or was in the stage before) become zeros; values that only some rows must not see are
      // taken out of the tile, and added to the rows that do see them.
      uint4* const chunks = reinterpret_cast<uint4*>(smem + (v_s - smem_u32(smem)));
      auto odd_chunk = [](const uint4& v) { return odd_word<T>(v.x) | odd_word<T>(v.y) | odd_word<T>(v.z) | odd_word<T>(v.w); };
      uint32_t odd = 0;
#pragma unroll 8
      for (int i = lane; i < KT * CH; i += 32) odd |= odd_chunk(chunks[i]);
      bool any = __any_sync(0xffffffffu, odd != 0);
      if (any) {
        odd = 0;
#pragma unroll 1
        for (int i = lane; i < KT * CH; i += 32) {
          if ((valid >> ((i >> 3) & (KT - 1))) & 1) odd |= odd_chunk(chunks[i]);
          else chunks[i] = make_uint4(0, 0, 0, 0);
        }
        any = __any_sync(0xffffffffu, odd != 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // TMA writes the stage next
        __syncwarp();
      }
      if (any) {
        T* vt = reinterpret_cast<T*>(smem + (v_s - smem_u32(smem)));
#pragma unroll
        for (int i = 0; i < DP / 8; i++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int d = 8 * i + cq + e;
#pragma unroll 1
            for (int key = 0; key < KT; key++) {
              const float v = to_f32(vt[swizzled(key, d >> 3) / 2 + (d & 7)]);
              if (fabsf(v) <= 3.4028235e38f || !((valid >> key) & 1)) continue;
              if (key0 + key < lim[0]) o[i][e] += v;
              if (key0 + key < lim[1]) o[i][2 + e] += v;
            }
          }
        __syncwarp();
#pragma unroll 1
        for (int i = lane; i < KT * DP; i += 32)
          if (!(fabsf(to_f32(vt[i])) <= 3.4028235e38f)) vt[i] = from_f32<T>(0.0f);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // TMA writes the stage next
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
    if (tile + 1 < tile1 && ok) load(next, at[turn ^ 1], true);
    else asm volatile("cp.async.commit_group;" ::: "memory");
    if (tile + 1 == tile1 || at[turn ^ 1].t == 0) {
      // The part's share of the segment ends here.
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
      }
      if (!ok) l0 = l1 = __uint_as_float(0x7fc00000u);
      const int id = pl.segs[c.b] + c.mb * H + c.g;
      const bool first = tile - c.t >= tile0, last = c.t + 1 == c.nt;  // of the segment's parts
      if (lane == 0) {
        if (first) p.seg_parts[id].x = w;
        if (last) p.seg_parts[id].y = w;
      }
      if (ALONE && first && last && c.b < B && !(pl.len[B] && sees_prefix(p, pl, c.b))) {
        // All that there is for these rows: the result itself, by the joining kernel's arithmetic.
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int r = r0 + 8 * h, row = c.mb * kRows + r, tok = p.by_group(row);
          if (r >= rows_in) continue;
          const float l = h ? l1 : l0, m = h ? m1 : m0, inv = l == 0.0f ? 0.0f : 1.0f / l;
          const int64_t token = pl.q0[c.b] + tok, head = c.g * p.group + row - tok * p.group;
          T* out = static_cast<T*>(p.a.out) + token * p.a.o_tok + head * p.a.o_head;
#pragma unroll
          for (int i = 0; i < DP / 8; i++) {
            const int d = 8 * i + cq;
            if (d < D) store_pair<T>(p, out + d, o[i][2 * h] * inv, o[i][2 * h + 1] * inv);
          }
          if (p.a.lse && (lane & 3) == 0) p.a.lse[token * p.a.lse_tok + head] = lse_of(m, l);
        }
      } else {
        float* slot = p.part + (int64_t)(w + id) * (kRows * (DP + 2));
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
    __syncwarp();
    if (tile + 2 < tile1) {
      step(turn ^ 1, turn);
      page = ask(at[turn]);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace
}  // namespace vtq
