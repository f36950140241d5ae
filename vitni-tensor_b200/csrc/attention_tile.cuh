// attention_tile.cuh -- attention_paged: the shared prefix on tcgen05.
//
// A CTA runs STREAMS streams of one softmax warpgroup each over a run of key tiles. With RT = 2 the
// streams are two blocks of 128 query rows that share every key tile; with RT = 1 they are the even and
// the odd key tiles of one block (two parts of the same rows, joined later), so that a stream's softmax
// runs beside the other's products. (S twice for each stream, with tiles of 64 keys for TMEM's sake, is
// slower: an MMA of 64 columns takes as long as one of 128, 5600 cycles a 256 x 128 step.)
//   softmax warpgroups  the query rows of a segment; then a thread a row: S from TMEM, the weights back into
//                       TMEM as the second product's A
//   2 loader warps      pages into a ring of swizzled K and V tiles, by TMA where a page holds 4 positions
//                       or more (gathering rows with 16-byte copies took three warps 5700 cycles a tile)
//   a warp a stream     one thread issues S = Q K^T (N = KT keys) and O += P V (V as it lies: N-major)
// O stays in TMEM; it is scaled again only where a row's maximum has grown by more than 2^8 (f16: 2^4) since the
// last time, until then the weights are taken relative to the old one (at most 256, and l with them; Weights).
// Head dims over 128 have room in TMEM for one stream.
#pragma once
#include "attention_plan.cuh"

namespace vtq {
namespace {

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
  static constexpr size_t SMEM = Q_BYTES + NSLOT * SLOT;
};
constexpr int kLoaders = 2, kMasks = 8;
static_assert(2 * kMasks > 14 + 1, "a mask's place must not come round before its tile's V slot has");

// The role of CTA `cta` of `ctas`.
template <typename T, int DP, int KT, int RT, int STREAMS, int NSLOT>
__device__ __forceinline__ void tile_role(const AttnParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv, uint8_t* gbase,
                                          int cta, int ctas) {
  using L = TileShape<T, DP, KT, RT, STREAMS, NSLOT>;
  constexpr uint32_t kFmt = std::is_same<T, __half>::value ? 0u : 1u;
  constexpr uint32_t kIdescS = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((uint32_t)(KT >> 3) << 17) | (8u << 24);
  constexpr uint32_t kIdescO = (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | (8u << 24);
  constexpr int TPS = STREAMS / RT;   // key tiles of a step: 2 where the streams are the tiles
  constexpr uint32_t kColO = STREAMS * KT;  // columns: each stream's S / P, then each stream's O
  constexpr int kGroups = KT / 4;     // of 4 keys: loader lw copies groups lw, lw + 3, ..
  static_assert(STREAMS * (KT + DP) <= 512 && NSLOT <= 14 && RT <= STREAMS, "TMEM, masks");
  __shared__ __align__(8) uint64_t s_bar[2 * NSLOT + 12 + kMasks];
  __shared__ uint32_t s_valid[kMasks][kLoaders][2];
  __shared__ uint32_t s_slot;
  __shared__ int s_abort;
  const uint32_t base = smem_u32(gbase), ring = base + L::Q_BYTES;
  auto bar = [&](int i) { return smem_u32(&s_bar[i]); };
  auto FULL = [&](int s) { return bar(s); };
  auto EMPTY = [&](int s) { return bar(NSLOT + s); };
  auto S_FULL = [&](int r) { return bar(2 * NSLOT + r); };              // of a stream
  auto P_FULL = [&](int r, int h) { return bar(2 * NSLOT + 2 + 2 * r + h); };  // of its P's two halves
  auto PV_DONE = [&](int r) { return bar(2 * NSLOT + 6 + r); };
  const uint32_t Q_FULL = bar(2 * NSLOT + 8), Q_EMPTY = bar(2 * NSLOT + 9);
  auto TURN = [&](int r) { return bar(2 * NSLOT + 10 + r); };  // stream r may take its exponentials
  auto MASK = [&](int i) { return bar(2 * NSLOT + 12 + i); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int D = (int)p.a.kv.head_dim;
  volatile int* abort_flag = &s_abort;

  if (tid == 0) {
    for (int s = 0; s < NSLOT; s++) {
      tc5::bar_init(FULL(s), 32 * kLoaders);
      tc5::bar_init(EMPTY(s), STREAMS / TPS);  // the streams that share a tile
    }
    for (int r = 0; r < 2; r++) {
      tc5::bar_init(S_FULL(r), 1);
      for (int h = 0; h < 2; h++) tc5::bar_init(P_FULL(r, h), 128);
      tc5::bar_init(PV_DONE(r), 1);
      tc5::bar_init(TURN(r), 128);
    }
    tc5::bar_init(Q_FULL, 128 * STREAMS);
    tc5::bar_init(Q_EMPTY, STREAMS);
    for (int i = 0; i < kMasks; i++) tc5::bar_init(MASK(i), kLoaders);
    *abort_flag = 0;
    fence_mbar_init();
  }
  constexpr int kMmaWarp = 4 * STREAMS + kLoaders;  // of stream 0
  if (warp == kMmaWarp) tc5::alloc(smem_u32(&s_slot), 512);
  tc5::fence_before();
  __syncthreads();
  tc5::fence_after();
  const uint32_t tmem = s_slot;
  // Steps [step0, step1) of all segments; a segment is (kv head g, block of RT x 128 rows).
  const int step0 = first_tile(p.tiles_total, ctas, cta), steps = first_tile(p.tiles_total, ctas, cta + 1) - step0;
  const int each = p.tiles_each, rows = (int)p.a.tokens * p.group;
  auto fail = [&]() {
    if (p.a.status) atomicOr(p.a.status, KERR_TIMEOUT);
    *abort_flag = 1;
  };
  // Whether stream r has rows in a segment.
  auto live = [&](int seg, int r) { return RT == 1 || ((seg % p.tile_segs) * RT + r) * kTileRows < rows; };
  // Word w of loader lw's part of s_valid where every key is there.
  auto full_word = [](int lw, int w) {
    const int keys = 4 * ((kGroups - lw + kLoaders - 1) / kLoaders) - 32 * w;
    return keys >= 32 ? 0xffffffffu : keys > 0 ? (1u << keys) - 1u : 0u;
  };
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
      const int box = p.box, boxes = box ? KT / box : 0;  // keys of a TMA box, boxes of a tile (32 at most)
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
      auto page_at = [&](int pos) { return pos < p.prefix ? p.a.kv.table[p.by_page(pos)] : -1; };
      int seg = step0 / each, kt = (step0 - seg * each) * TPS;
      int g = seg / p.tile_segs;
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
                s_valid[n % kMasks][lw][w] = full_word(lw, w);
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
              const int slot = box_pos - p.by_page(box_pos) * page_size;
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
            const int64_t slot = pos - p.by_page(pos) * page_size;
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
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      if (ok && !*abort_flag) tell(2 * tiles);
      else if (lane == 0) fail();
    } else {
      // ---- products of stream r ----
      // (One warp that looks after both streams finds each barrier some 500 cycles late; 6600 cycles a step.)
      const int r = warp - kMmaWarp;
      const uint32_t one = tc5::elect(), S = tmem + r * KT, O = tmem + kColO + r * DP;
      int k_at = TPS == 2 ? 2 * r : 0, v_at = k_at + 1;  // ring places of this step's K and V, and their phases
      uint32_t k_ph = 0, v_ph = 0, q_ph = 0, used = 0;   // used: of the stream's own barriers
      int in = step0 % each, mt = step0 / each % p.tile_segs;
      bool ok = true, used_before = false;
      for (int i = 0; i < steps && r < STREAMS; i++) {
        const bool fresh = i == 0 || in == 0, last_of_q = i + 1 == steps || in + 1 == each;
        const bool on = RT == 1 || (mt * RT + r) * kTileRows < rows;
        if (fresh) {
          ok = tc5::bar_wait(Q_FULL, q_ph);
          q_ph ^= 1;
        }
        ok = ok && tc5::bar_wait(FULL(k_at), k_ph);
        if (!on) {
          // No rows: it only takes its part in the releases, each place once it has been filled.
          if (lane == 0 && ok) {
            tc5::bar_arrive(EMPTY(k_at));
            if (last_of_q) tc5::bar_arrive(Q_EMPTY);
          }
          ok = ok && tc5::bar_wait(FULL(v_at), v_ph);
          if (lane == 0 && ok) tc5::bar_arrive(EMPTY(v_at));
        } else {
          // S takes the place of the P before it, whose product has to be done by then, not only asked for:
          // MMAs with other accumulators need not run in the order of their issue.
          if (used_before) ok = ok && tc5::bar_wait(PV_DONE(r), used ^ 1);
          if (!ok) break;
          __syncwarp();
          tc5::fence_after();
          const uint32_t q_s = base + (RT == 2 ? r : 0) * L::Q_TILE, k_s = ring + k_at * L::SLOT, v_s = ring + v_at * L::SLOT;
#pragma unroll
          for (int k = 0; k < DP / 16; k++)
            mma_ss(S, tc5::desc_sw128(q_s + (k >> 2) * (kTileRows * 128) + (k & 3) * 32),
                   tc5::desc_sw128(k_s + (k >> 2) * (KT * 128) + (k & 3) * 32), kIdescS, k > 0, one);
          tc5::commit(S_FULL(r), one);
          tc5::commit(EMPTY(k_at), one);
          if (last_of_q) tc5::commit(Q_EMPTY, one);
          ok = tc5::bar_wait(FULL(v_at), v_ph);
#pragma unroll
          for (int h = 0; h < 2; h++) {
            ok = ok && tc5::bar_wait(P_FULL(r, h), used);
            if (!ok) break;
            __syncwarp();
            tc5::fence_after();
#pragma unroll
            for (int k = 0; k < KT / 32; k++)
              mma_ts(O, S + 8 * (h * (KT / 32) + k), desc_n_major(v_s + (h * (KT / 32) + k) * 2048, KT * 128), kIdescO,
                     !(fresh && h == 0 && k == 0), one);
          }
          if (!ok) break;
          tc5::commit(PV_DONE(r), one);
          tc5::commit(EMPTY(v_at), one);
          used ^= 1;
          used_before = true;
        }
        if (!ok) break;
        if ((k_at += 2 * TPS) >= NSLOT) k_at -= NSLOT, k_ph ^= 1;
        if ((v_at += 2 * TPS) >= NSLOT) v_at -= NSLOT, v_ph ^= 1;
        if (++in == each) {
          in = 0;
          if (++mt == p.tile_segs) mt = 0;
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
    int had = 0;                    // segments that this CTA is done with
    // The query rows of a segment, by all softmax warps, 8 lanes a row of 128 bytes: the first ones while the first
    // keys are on their way (5.8 us where the two loaders brought them), the next ones behind a segment's last weights.
    auto ask_q = [&](int s) {
      const int g = s / p.tile_segs, row0 = (s - g * p.tile_segs) * RT * kTileRows;
#pragma unroll 4
      for (int i = warp * 4 + (lane >> 3); i < RT * kTileRows; i += 16 * STREAMS) {
        const int q = row0 + i, tok = p.by_group(q);
        const bool in = q < rows;
        const T* src = static_cast<const T*>(p.a.q) + (in ? (int64_t)tok * p.a.q_tok + (int64_t)(g * p.group + q - tok * p.group) * p.a.q_head : 0);
#pragma unroll
        for (int c = 0; c < DP / 64; c++) {
          const int chunk = c * 8 + (lane & 7);
          const bool there = in && chunk * 8 < D;
          const uint32_t at = (i / kTileRows) * L::Q_TILE + place(kTileRows, i % kTileRows, chunk);
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
    };
    auto tell_q = [&]() {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc5::bar_arrive(Q_FULL);
    };
    // Every product with this segment's queries is done: the next segment's may take their place.
    auto next_q = [&](int s) {
      if (!tc5::bar_wait(Q_EMPTY, tc5::phase(had++, 1))) return false;
      ask_q(s);
      return true;
    };
    if (steps) {
      ask_q(step0 / each);
      tell_q();
    }
    int seg = step0 / each, in = step0 - seg * each, i = 0;
    for (; i < steps; i++) {
      const bool start = i == 0 || in == 0, last = i + 1 == steps || in + 1 == each;
      const int this_seg = seg;
      if (++in == each) in = 0, seg++;
      // The streams take turns at their exponentials, stream 0 first, one beginning when the other is half
      // through: left alone they fall into step, and both wait for the exponential unit, then both for the
      // tensor cores (4700 cycles a step).
      const uint32_t turn = (uint32_t)(i - (r == 0)) & 1u;
      const bool wait_turn = STREAMS == 2 && (r == 1 || i > 0);
      if (!live(this_seg, r)) {
        if (wait_turn && !tc5::bar_wait(TURN(r), turn)) {
          if (lane == 0) fail();
          break;
        }
        if (STREAMS == 2) tc5::bar_arrive(TURN(1 - r));
        if (last && i + 1 < steps) {
          if (!next_q(this_seg + 1)) {
            if (lane == 0) fail();
            break;
          }
          tell_q();
        }
        continue;
      }
      const int n = i * TPS + (TPS == 2 ? r : 0);
      const uint32_t sp = tmem + lanes + r * KT;
      bool whole = tc5::bar_wait(MASK(n % kMasks), tc5::phase(n, kMasks));
      if (!whole || !tc5::bar_wait(S_FULL(r), used & 1)) {
        if (lane == 0) fail();
        break;
      }
      tc5::fence_after();
      // The row is read twice, a half at a time, in loops that stay in the instruction cache: the same
      // arithmetic unrolled over a whole row waits more for instructions than for anything else (2.4 of
      // 4 cycles an instruction).
#pragma unroll
      for (int w = 0; w < kLoaders; w++) {
        const uint32_t lo = full_word(w, 0), hi = full_word(w, 1);
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
      constexpr int HALF = KT / 2;  // columns at a time: a half of P
      float top;
      {
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 2; c++) {
          float x[HALF];
#pragma unroll
          for (int j = 0; j < HALF; j += 32) tmem_ld32(sp + c * HALF + j, x + j);
          tc5::wait_ld();
#pragma unroll
          for (int j = 0; j < HALF; j += 4) {
            t0 = fmaxf(fmaxf(x[j], x[j + 1]), t0);
            t1 = fmaxf(fmaxf(x[j + 2], x[j + 3]), t1);
          }
        }
        top = Weights<T>::base(fmaxf(t0, t1), p.scale_log2, Weights<T>::tile_up);
      }
      if (p.scale_log2 < 0.0f) {  // the largest score is that of the smallest product
        float low = INFINITY;
#pragma unroll 1
        for (int c = 0; c < KT / 32; c++) {
          float z[32];
          tmem_ld32(sp + 32 * c, z);
          tc5::wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j++) low = fminf(low, z[j]);
        }
        top = Weights<T>::base(low, p.scale_log2, Weights<T>::tile_up);
      }
      if (start) {
        m = top;
        l = 0.0f;
      } else {
        const bool grow = top - m > Weights<T>::tile_grow;  // (both -inf: not; m alone: it is)
        if (__any_sync(0xffffffffu, grow)) {
          const float to = grow ? top : m;
          const float f = !grow ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast(m - to);
          // (This S was asked for when the product before it was done.)
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
      if (wait_turn && !tc5::bar_wait(TURN(r), turn)) {
        if (lane == 0) fail();
        break;
      }
      // P in the place of S: 16 columns for 32, so that a chunk never lands on columns not read yet.
      const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), u2 = make_float2(-u, -u);
      float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
      float x[HALF];
#pragma unroll
      for (int j = 0; j < HALF; j += 32) tmem_ld32(sp + j, x + j);
#pragma unroll 1
      for (int c = 0; c < 2; c++) {
        tc5::wait_ld();
        float2 e[HALF / 2];
#pragma unroll
        for (int j = 0; j < HALF / 2; j++) e[j] = fma2(make_float2(x[2 * j], x[2 * j + 1]), scale2, u2);
        if (c == 0) {
#pragma unroll
          for (int j = 0; j < HALF; j += 32) tmem_ld32(sp + HALF + j, x + j);
        }
        uint32_t w[HALF / 2];
#pragma unroll
        for (int j = 0; j < HALF / 2; j++) {
          e[j].x = exp2_fast(e[j].x);
          e[j].y = exp2_fast(e[j].y);
          if (j & 1) sum1 = add2(sum1, e[j]);
          else sum0 = add2(sum0, e[j]);
          w[j] = pack2<T>(e[j].x, e[j].y);
        }
#pragma unroll
        for (int j = 0; j < HALF / 2; j += 16) tmem_st16(sp + c * (HALF / 2) + j, w + j);
        // This half's product can start.
        tmem_wait_st();
        tc5::fence_before();
        tc5::bar_arrive(P_FULL(r, c));
        if (STREAMS == 2 && c == 0) tc5::bar_arrive(TURN(1 - r));
      }
      l += (sum0.x + sum0.y) + (sum1.x + sum1.y);
      used++;
      if (last) {
        if ((i + 1 < steps && !next_q(this_seg + 1)) || !tc5::bar_wait(PV_DONE(r), (used - 1) & 1)) {
          if (lane == 0) fail();
          break;
        }
        tc5::fence_after();
        float* slot = p.tile_part + (int64_t)((cta + this_seg) * STREAMS + r) * (kTileRows * (DP + 2));
        if (tid == 0) {
          const int done = step0 + i - this_seg * each;  // this step's place in the segment
          if (done <= i) p.seg_ctas[this_seg].x = cta;   // its first step is among this CTA's
          if (done + 1 == each) p.seg_ctas[this_seg].y = cta;
        }
        const bool there = ((this_seg % p.tile_segs) * RT + (RT == 2 ? r : 0)) * kTileRows + row < rows;
        if (there) *reinterpret_cast<float2*>(slot + 2 * row) = make_float2(m, l);
#pragma unroll 1
        for (int c = 0; c < DP / 32; c++) {
          float o[32];
          tmem_ld32(so + 32 * c, o);
          tc5::wait_ld();
          if (there) {
            float* dst = slot + 2 * kTileRows + row * DP + 32 * c;
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + j), "f"(o[j]), "f"(o[j + 1]),
                           "f"(o[j + 2]), "f"(o[j + 3]), "f"(o[j + 4]), "f"(o[j + 5]), "f"(o[j + 6]), "f"(o[j + 7])
                           : "memory");
          }
        }
        tc5::fence_before();
        if (i + 1 < steps) tell_q();
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // A wait ran out: the segments that this warp's rows have not left yet become NaN (their sums of weights are), so
    // that the joining kernel finds an entry and a slot for each of them, and rows that lack keys show it.
    if (i < steps) {
      for (int s = (step0 + i) / each; s <= (step0 + steps - 1) / each; s++) {
        if (tid == 0) {
          if (s * each >= step0) p.seg_ctas[s].x = cta;
          if ((s + 1) * each <= step0 + steps) p.seg_ctas[s].y = cta;
        }
        if (((s % p.tile_segs) * RT + (RT == 2 ? r : 0)) * kTileRows + row < rows)
          *reinterpret_cast<float2*>(p.tile_part + (int64_t)((cta + s) * STREAMS + r) * (kTileRows * (DP + 2)) + 2 * row) =
              make_float2(0.0f, __uint_as_float(0x7fc00000u));
      }
    }
  }
  if (*abort_flag) tc5::settle();
  tc5::fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc5::fence_after();
    tc5::dealloc(tmem, 512);
  }
}

}  // namespace
}  // namespace vtq
