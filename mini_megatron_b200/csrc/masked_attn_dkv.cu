// Masked attention backward, key side: dK and dV.
//
//   dV_j = sum_i P_ij dO_i,  dK_j = s sum_i dS_ij q_i   (P, dS: masked_attn_dq.cu)
//
// The sums run over every query that sees key j, in all heads that share the K/V
// head, in a fixed order in 32-bit TMEM accumulators: shared heads need no
// reduction afterwards and the result does not depend on scheduling.
//
// Persistent grid, one CTA per SM; a work item is (batch, K/V head, 128-row key
// tile).  Scores are computed transposed (a thread owns a key row), so P^T and dS^T
// go back into TMEM as the first operands of the two sums and never touch shared
// memory; LSE and Delta of the query rows arrive with the Q / dO tiles by bulk copies.
// The queries that see a key are an interval too (document_plan.cu), so a mask is two
// numbers per thread here as well.  Roles (20 warps):
//
//   warp 0     TMA: K_j, V_j per item; Q_i, dO_i and their row data into a ring
//   warp 1     TMEM allocation; one thread issues S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//   warp 2     hands out the work items
//   warp 3     stores finished dK / dV tiles from the Q / dO stage they were staged in
//   warps 4-19 softmax gradient: four warps share 32 key rows, each has 32 of the 128 queries
//              (masked_attn_dq.cu says why four; with two 100 us instead of 96 at 16 x 1024 tokens, 12 heads of 64)
//
// d = 64: S^T has two TMEM buffers, the next tile's scores are computed while this tile's
// softmax runs.  d = 128: S^T, dP^T, dV and dK fill TMEM; the next S^T follows dV and the next
// dP^T follows dK, each overlapping the other half of the softmax gradient.
//
// What bounds it, causal rows: as in masked_attn_dq.cu, with four products a tile.  16 x 1024 tokens, 12 heads of
// 64: 75.5 us, 770 TFLOP/s over the tiles visited; 16384 tokens, 8 heads of 128: 836 us, 1330 TFLOP/s.
#include "masked_attn.cuh"

namespace mmb {
namespace mattn {
namespace dkv {

constexpr int kThreads = 640;
constexpr int kWarps = 16;  // of the softmax gradient

template <int D>
struct Cfg {
  static constexpr int TILE = BT * D * 2;
  static constexpr int KB = (D == 64) ? 2 : 1;  // K / V buffers
  static constexpr int NQ = (D == 64) ? 4 : 2;  // Q / dO ring stages
  static constexpr int SB = (D == 64) ? 2 : 1;  // S^T buffers in TMEM
  // dK and dV of an item leave during the next item's first pair.  d = 128: they leave at once, with two stages the one
  // they are staged in is needed again by then.
  static constexpr bool DEFER = (D == 64);
  static constexpr int K_OFF = 0;               // [KB][K, V]
  static constexpr int Q_OFF = KB * 2 * TILE;   // [NQ][Q, dO]
  static constexpr int LD_OFF = Q_OFF + NQ * 2 * TILE, LD = 1024;  // [NQ][-LSE log2 e 128, -Delta 128]
  static constexpr int ITEM_OFF = LD_OFF + NQ * LD;  // [kRing] work items
  static constexpr int BAR_OFF = ITEM_OFF + kRing * 32;
  static constexpr int SMEM = 1024 + BAR_OFF + 384;
  static constexpr uint32_t T_S = 0, T_DP = SB * 128, T_DV = T_DP + 128, T_DK = T_DV + D;
};
static_assert(Cfg<128>::SMEM <= 227 * 1024 && Cfg<64>::SMEM <= 227 * 1024, "shared memory of one CTA");
static_assert(Cfg<128>::T_DK + 128 <= 512 && Cfg<64>::T_DK + 64 <= 512, "TMEM columns");

struct Args {
  int B, S, nh, nkv, n_t;
  int parts, heads;     // an item's share: `heads` = nh / nkv / parts query heads
  FastDiv by_parts, by_nkv, by_B, by_tiles;
  Mask mask;
  const float* slopes;
  Score score;
  float scale;
  const float* ld;      // [B, nh, n_t, 2, 128]
  __nv_bfloat16* dqkv;  // [B, S, (nh + 2 nkv) * D]
  float* partial;       // parts > 1: [parts, B, S, 2 nkv * D] sums of each share
  int* err;
};

struct alignas(16) Item {
  int b, hk, t;  // b < 0: no more items
  int part;      // which share of the K/V head's query heads
  int2 r, f;     // query tiles, and those of them that need no mask
};
static_assert(sizeof(Item) <= 32, "ring entry");
constexpr int kConsumers = 1 + 1 + 1 + kWarps;  // TMA and MMA threads, store and softmax warps

__device__ __forceinline__ Item decode(const Args& a, int item) {
  const int q = a.by_parts.quot(item);
  const int li = a.by_nkv.quot(q);
  Item it;
  it.part = item - q * a.parts;
  it.hk = q - li * a.nkv;
  if (a.mask.order) {
    const int e = ordered(a.mask.order, li, a.B * a.n_t);
    it.b = a.by_tiles.quot(e);
    it.t = e - it.b * a.n_t;
  } else {  // causal rows: the first key tile is seen by the most queries
    it.t = a.by_B.quot(li);
    it.b = li - it.t * a.B;
  }
  query_tiles(a.mask, it.b, a.n_t, it.t, it.r, it.f);
  return it;
}

// 32 bytes of one row.
__device__ __forceinline__ void store8(float* p, const uint32_t* v, float mul) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(__uint_as_float(v[0]) * mul),
               "f"(__uint_as_float(v[1]) * mul), "f"(__uint_as_float(v[2]) * mul), "f"(__uint_as_float(v[3]) * mul),
               "f"(__uint_as_float(v[4]) * mul), "f"(__uint_as_float(v[5]) * mul), "f"(__uint_as_float(v[6]) * mul),
               "f"(__uint_as_float(v[7]) * mul)
               : "memory");
}

// (head of the item's share, query tile) pairs of this CTA's items, one after another.
struct Walk {
  int it = -1, g = 0, i = 0;
  Item w;
  // 1: at the next pair, 0: no more, -1: the wait for an item ran out
  __device__ __forceinline__ int next(const Ring<Item>& ring, int heads, int* err, volatile int* abort_flag) {
    if (it >= 0) {
      if (++i < w.r.y) return 1;
      if (++g < heads) {
        i = w.r.x;
        return 1;
      }
    }
    if (!ring.get_thread(w, ++it, err, abort_flag)) return -1;
    g = 0;
    i = w.r.x;
    return w.b >= 0;
  }
  __device__ __forceinline__ bool first() const { return g == 0 && i == w.r.x; }
  __device__ __forceinline__ bool last(int heads) const { return g == heads - 1 && i == w.r.y - 1; }
};

template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
    masked_attn_dkv_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_do,
                           const __grid_constant__ CUtensorMap tm_dqkv, const Args a) {
  pdl_trigger();
  using C = Cfg<D>;
  constexpr int KB = C::KB, NQ = C::NQ, SB = C::SB;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sKV = smem + C::K_OFF;
  uint8_t* sQ = smem + C::Q_OFF;
  uint8_t* sLD = smem + C::LD_OFF;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* k_full = bars;         // [2]
  uint64_t* k_empty = bars + 2;    // [2]
  uint64_t* v_full = bars + 4;     // [2]
  uint64_t* v_empty = bars + 6;    // [2]
  uint64_t* q_full = bars + 30;    // [4]
  uint64_t* q_empty = bars + 34;   // [4]
  uint64_t* s_full = bars + 10;    // [2]
  uint64_t* dp_full = bars + 12;
  // P^T written, S^T read (16 warps).  Two barriers: a warp may be done with P^T(n+1) before another one is
  // with P^T(n), and its second arrival must not complete the first one's phase.
  uint64_t* p_full = bars + 18;    // [2]
  uint64_t* ds_full = bars + 14;   // dS^T written, dP^T and the row data read (16 warps)
  uint64_t* g_full = bars + 15;    // dK, dV of an item complete
  uint64_t* g_free = bars + 16;    // ... read (16 warps)
  uint64_t* drain = bars + 17;
  uint64_t* out_full = bars + 20;  // dK, dV of an item staged (16 warps)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 38);  // bars + 21 ..: the ring of work items
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Ring<Item> ring{reinterpret_cast<Item*>(smem + C::ITEM_OFF), bars + 21, bars + 21 + kRing};
  const int heads = a.heads;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kWarps);
    }
    for (int i = 0; i < NQ; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&bars[21 + i], 1);
      mbar_init(&bars[21 + kRing + i], kConsumers);
    }
    mbar_init(dp_full, 1);
    mbar_init(ds_full, kWarps);
    mbar_init(g_full, 1);
    mbar_init(g_free, kWarps);
    mbar_init(out_full, kWarps);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tm_qkv);
    prefetch_tmap(&tm_do);
    prefetch_tmap(&tm_dqkv);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    reg_dec<64>();
    if (warp == 0) {
      if (elect_one()) {
        // ---------------------------------------------------------------- TMA
        int n = 0, k_issued = -1, v_issued = -1;
        bool ok = true;
        Walk x;
        for (int got; (got = x.next(ring, heads, a.err, abort_flag)) != 0; ++n) {
          if (got < 0) { ok = false; break; }
          if (x.first()) {
            const int kb = x.it % KB;
            uint8_t* kd = sKV + kb * 2 * C::TILE;
            if (x.it >= KB && !bwait(&k_empty[kb], ((x.it / KB) - 1) & 1, a.err, abort_flag)) { ok = false; break; }
            mbar_expect_tx(&k_full[kb], C::TILE);
            load_tile<D>(kd, &tm_qkv, &k_full[kb], (a.nh + x.w.hk) * D, x.w.t * BT, x.w.b);
            k_issued = x.it;
            if (x.it >= KB && !bwait(&v_empty[kb], ((x.it / KB) - 1) & 1, a.err, abort_flag)) { ok = false; break; }
            mbar_expect_tx(&v_full[kb], C::TILE);
            load_tile<D>(kd + C::TILE, &tm_qkv, &v_full[kb], (a.nh + a.nkv + x.w.hk) * D, x.w.t * BT, x.w.b);
            v_issued = x.it;
          }
          const int st = n % NQ;
          if (n >= NQ && !bwait(&q_empty[st], ((n / NQ) - 1) & 1, a.err, abort_flag)) { ok = false; break; }
          const int h = (x.w.hk * a.parts + x.w.part) * heads + x.g;
          mbar_expect_tx(&q_full[st], 2 * C::TILE + 1024);
          load_tile<D>(sQ + st * 2 * C::TILE, &tm_qkv, &q_full[st], h * D, x.i * BT, x.w.b);
          load_tile<D>(sQ + st * 2 * C::TILE + C::TILE, &tm_do, &q_full[st], h * D, x.i * BT, x.w.b);
          bulk_load(sLD + st * C::LD, a.ld + (((size_t)x.w.b * a.nh + h) * a.n_t + x.i) * (2 * BT), 1024, &q_full[st]);
        }
        if (!ok) {
          for (int u = max(0, k_issued - KB + 1); u <= k_issued; ++u) drain_wait(&k_full[u % KB], (u / KB) & 1);
          for (int u = max(0, v_issued - KB + 1); u <= v_issued; ++u) drain_wait(&v_full[u % KB], (u / KB) & 1);
          for (int u = max(0, n - NQ); u < n; ++u) drain_wait(&q_full[u % NQ], (u / NQ) & 1);
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      if (elect_one()) {
        // ---------------------------------------------------------------- MMA
        bool ok = true;
        int n = 0;
        Walk cur, nxt;
        // K is only read by S^T and V only by dP^T: after an item's last one the next item's tile may load
        auto issue_s = [&](const Walk& x, int u) -> bool {
          const int kb = x.it % KB;
          if (x.first() && !bwait(&k_full[kb], (x.it / KB) & 1, a.err, abort_flag)) return false;
          if (!bwait(&q_full[u % NQ], (u / NQ) & 1, a.err, abort_flag)) return false;
          tc_fence_after();
          mma_abt<D>(tmem + C::T_S + (u % SB) * 128, smem_u32(sKV + kb * 2 * C::TILE),
                     smem_u32(sQ + (u % NQ) * 2 * C::TILE));
          umma_commit(&s_full[u % SB]);
          if (x.last(heads)) umma_commit(&k_empty[kb]);
          return true;
        };
        auto issue_dp = [&](const Walk& x, int u) -> bool {
          const int kb = x.it % KB;
          if (x.first() && !bwait(&v_full[kb], (x.it / KB) & 1, a.err, abort_flag)) return false;
          tc_fence_after();
          mma_abt<D>(tmem + C::T_DP, smem_u32(sKV + kb * 2 * C::TILE + C::TILE),
                     smem_u32(sQ + (u % NQ) * 2 * C::TILE + C::TILE));
          umma_commit(dp_full);
          if (x.last(heads)) umma_commit(&v_empty[kb]);
          return true;
        };
        int more = nxt.next(ring, heads, a.err, abort_flag);
        ok = more >= 0 && (more == 0 || (issue_s(nxt, 0) && issue_dp(nxt, 0)));
        while (ok && more) {
          cur = nxt;
          more = nxt.next(ring, heads, a.err, abort_flag);
          if (more < 0) { ok = false; break; }
          const uint32_t q_addr = smem_u32(sQ + (n % NQ) * 2 * C::TILE);
          if (SB == 2 && more && !issue_s(nxt, n + 1)) { ok = false; break; }
          if (!bwait(&p_full[n & 1], (n >> 1) & 1, a.err, abort_flag)) { ok = false; break; }
          if (cur.first() && cur.it > 0 && !bwait(g_free, (cur.it - 1) & 1, a.err, abort_flag)) { ok = false; break; }
          tc_fence_after();
          mma_tmem_b<D, 32>(tmem + C::T_DV, tmem + C::T_S + (n % SB) * 128, q_addr + C::TILE, !cur.first());
          if (SB == 1 && more && !issue_s(nxt, n + 1)) { ok = false; break; }  // over P^T, in issue order after dV
          if (!bwait(ds_full, n & 1, a.err, abort_flag)) { ok = false; break; }
          tc_fence_after();
          mma_tmem_b<D, 32>(tmem + C::T_DK, tmem + C::T_DP, q_addr, !cur.first());
          // the Q / dO stage of an item's last pair becomes the staging tile of its dK and dV, which releases it
          if (cur.last(heads)) umma_commit(g_full);
          else umma_commit(&q_empty[n % NQ]);
          if (more && !issue_dp(nxt, n + 1)) { ok = false; break; }  // over dS^T, in issue order after dK
          ++n;
        }
        if (!ok) {
          umma_commit(drain);
          drain_wait(drain, 0);
        }
      }
      __syncwarp();
    } else if (warp == 2) {
      // ---------------------------------------------------------------- work items
      // Only items with work travel through the ring: the MMA thread takes the next item before the other roles have
      // finished the current one, so a run of empty ones could fill the ring with nobody left to empty it.
      const int n_items = a.B * a.nkv * a.n_t * a.parts;
      Item w;
      for (int r = 0, k = 0;; ++r) {
        const int item = snake_item(r);
        if (item < n_items) {
          w = decode(a, item);
          if (w.r.x >= w.r.y) {
            const int rows = min(BT, a.S - w.t * BT);
            const size_t tok = (size_t)w.b * a.S + w.t * BT;
            if (a.parts > 1) {
              const size_t width = (size_t)2 * a.nkv * D;
              float* p = a.partial + ((size_t)w.part * a.B * a.S + tok) * width + (size_t)w.hk * D;
              zero_rows<4 * D>(p, 4 * width, rows);
              zero_rows<4 * D>(p + (size_t)a.nkv * D, 4 * width, rows);
            } else {
              const size_t width = (size_t)(a.nh + 2 * a.nkv) * D;
              __nv_bfloat16* p = a.dqkv + tok * width + (size_t)(a.nh + w.hk) * D;
              zero_rows<2 * D>(p, 2 * width, rows);
              zero_rows<2 * D>(p + (size_t)a.nkv * D, 2 * width, rows);
            }
            continue;
          }
        } else {
          w.b = -1;
        }
        if (!ring.put_warp(w, k++, a.err, abort_flag) || w.b < 0) break;
      }
    } else {
      // ---------------------------------------------------------------- stores of staged dK / dV tiles
      int n = 0, it = 0;
      Item w;
      for (int u = 0; ring.get_warp(w, u, a.err, abort_flag) && w.b >= 0; ++u) {
        n += (w.r.y - w.r.x) * heads;
        if (!wwait(out_full, it & 1, a.err, abort_flag)) break;
        if (lane == 0) {
          const int qs = (n - 1) % NQ;
          if (a.parts == 1) {
            uint8_t* stg = sQ + qs * 2 * C::TILE;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              tma_store_3d(&tm_dqkv, stg + c * 16384, (a.nh + w.hk) * D + c * 64, w.t * BT, w.b);
              tma_store_3d(&tm_dqkv, stg + C::TILE + c * 16384, (a.nh + a.nkv + w.hk) * D + c * 64, w.t * BT, w.b);
            }
            bulk_commit();
            bulk_wait_read<0>();
          }
          mbar_arrive(&q_empty[qs]);
        }
        __syncwarp();
        ++it;
      }
      if (lane == 0) bulk_wait<0>();
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ softmax gradient, dK / dV store
    reg_inc<104>();
    const int part = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;  // key row within the tile (TMEM lane)
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const Score k = a.score;
    int n = 0, it = 0;
    bool ok = true;
    // a share's sums: dK and dV of this warp's columns, [parts, B, S, 2 nkv * D]
    auto share_row = [&](const Item& w) {
      return a.partial + (((size_t)w.part * a.B + w.b) * a.S + w.t * BT + row) * ((size_t)2 * a.nkv * D) +
             (size_t)w.hk * D + part * (D / 4);
    };
    // dK and dV of item number `of`, whose last pair was number `last`: TMEM -> the Q / dO stage of that pair, for the
    // store warp, or, where they are a share's, to `pk` (nullptr: the row lies behind the end)
    auto drain_dkv = [&](int of, int last, float* pk) -> bool {
      if (!wwait(g_full, of & 1, a.err, abort_flag)) return false;
      tc_fence_after();
      uint32_t v[D / 4], u[D / 4];
      tmem_ld(tmem + C::T_DV + lane_off + part * (D / 4), v);
      tmem_ld(tmem + C::T_DK + lane_off + part * (D / 4), u);
      tmem_wait_ld();
      warp_arrive(g_free);
      if (a.parts > 1) {
        if (pk) {
#pragma unroll
          for (int c = 0; c < D / 4; c += 8) {
            store8(pk + c, &u[c], a.scale);
            store8(pk + (size_t)a.nkv * D + c, &v[c], 1.f);
          }
        }
      } else {
        uint8_t* stg = sQ + (last % NQ) * 2 * C::TILE;
        stage_row(stg, 16384, row, part * (D / 4), u, a.scale);
        stage_row(stg + C::TILE, 16384, row, part * (D / 4), v, 1.f);
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(out_full);
      return true;
    };
    int last_pair = -1;  // last pair of the item whose dK and dV are still in TMEM
    float* last_pk = nullptr;
    Item w;
    for (int u = 0; ok && (ok = ring.get_warp(w, u, a.err, abort_flag)) && w.b >= 0; ++u) {
      const int key = w.t * BT + row;
      const bool in = key < a.S;
      int first = key, last = a.n_t * BT;
      if (a.mask.rows) {
        const int* tr = a.mask.rows + ((size_t)w.b * a.n_t + w.t) * (4 * BT) + 2 * BT + row;
        first = tr[0];
        last = tr[BT];
      }
      for (int g = 0; ok && g < heads; ++g) {
        float slope = 0.f;
        if (BIAS) slope = a.slopes[(w.hk * a.parts + w.part) * heads + g] * kLog2e;
        for (int i = w.r.x; i < w.r.y; ++i, ++n) {
          const int st = n % NQ;
          const uint32_t t_s = tmem + C::T_S + (n % SB) * 128 + lane_off + part * 32;
          const uint32_t t_dp = tmem + C::T_DP + lane_off + part * 32;
          const float* l2 = reinterpret_cast<const float*>(sLD + st * C::LD) + part * 32;
          if (!wwait(&q_full[st], (n / NQ) & 1, a.err, abort_flag)) { ok = false; break; }
          if (!wwait(&s_full[n % SB], (n / SB) & 1, a.err, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const bool masked = i < w.f.x || i >= w.f.y;
          float pf[32];  // P (1 - tanh^2)
          {
            uint32_t s[32];
            tmem_ld(t_s, s);
            tmem_wait_ld();
            if (CAP) cap_in_place(s, k);
            const int q0 = i * BT + part * 32;  // query of column 0
            const uint32_t seen = masked ? seen_bits(first, last, q0) : 0xffffffffu;
            const float dist = (float)(q0 - key);
            uint32_t pp[16];
#pragma unroll
            for (int e4 = 0; e4 < 32; e4 += 4) {
              const float4 lv = *reinterpret_cast<const float4*>(l2 + e4);
#pragma unroll
              for (int u = 0; u < 4; u += 2) {
                const int e = e4 + u;
                float2 x = pair(s[e], s[e + 1]), f;
                const float2 ls = u == 0 ? make_float2(lv.x, lv.y) : make_float2(lv.z, lv.w);
                if (CAP) {
                  f = fma2(mul2(x, pair(-1.f)), x, pair(1.f));  // 1 - tanh^2
                  x = mul2(x, pair(k.cap));
                }
                if (BIAS) {
                  if (!CAP) x = mul2(x, pair(k.mul));
                  x.x = fmaf(-slope, fabsf(dist + (float)e), x.x);
                  x.y = fmaf(-slope, fabsf(dist + (float)(e + 1)), x.y);
                }
                x = (CAP || BIAS) ? add2(x, ls) : fma2(x, pair(k.mul), ls);
                x = exp2_pair(x);
                if (masked) {
                  if (!(seen & (1u << e))) x.x = 0.f;
                  if (!(seen & (2u << e))) x.y = 0.f;
                }
                pp[e / 2] = pack_bf16x2(x.x, x.y);
                if (CAP) x = mul2(x, f);
                pf[e] = x.x;
                pf[e + 1] = x.y;
              }
            }
            tmem_st_32x32b_x16(t_s, pp);  // over S^T columns already read
          }
          tmem_wait_st();
          warp_arrive(&p_full[n & 1]);
          // the previous item's dK and dV leave here: its last products ran while this pair's P was computed
          if (C::DEFER && last_pair >= 0) {
            if (!drain_dkv(it - 1, last_pair, last_pk)) { ok = false; break; }
            last_pair = -1;
          }
          if (!wwait(dp_full, n & 1, a.err, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const float* delta = l2 + BT;
          {
            uint32_t dp[32];
            tmem_ld(t_dp, dp);
            tmem_wait_ld();
            uint32_t ds[16];
#pragma unroll
            for (int e4 = 0; e4 < 32; e4 += 4) {
              const float4 dl = *reinterpret_cast<const float4*>(delta + e4);
              const float2 v = mul2(make_float2(pf[e4], pf[e4 + 1]), add2(pair(dp[e4], dp[e4 + 1]), make_float2(dl.x, dl.y)));
              const float2 z = mul2(make_float2(pf[e4 + 2], pf[e4 + 3]),
                                    add2(pair(dp[e4 + 2], dp[e4 + 3]), make_float2(dl.z, dl.w)));
              ds[e4 / 2] = pack_bf16x2(v.x, v.y);
              ds[e4 / 2 + 1] = pack_bf16x2(z.x, z.y);
            }
            tmem_st_32x32b_x16(t_dp, ds);  // over dP^T columns already read
          }
          tmem_wait_st();
          warp_arrive(ds_full);
        }
      }
      if (!ok) break;
      last_pair = n - 1;
      last_pk = a.parts > 1 && in ? share_row(w) : nullptr;
      ++it;
      if (!C::DEFER && !drain_dkv(it - 1, last_pair, last_pk)) { ok = false; break; }
    }
    if (C::DEFER && ok && last_pair >= 0) drain_dkv(it - 1, last_pair, last_pk);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool CAP, bool BIAS>
int launch(const CUtensorMap& tq, const CUtensorMap& to, const CUtensorMap& td, const Args& a, int grid, cudaStream_t stream) {
  auto k = masked_attn_dkv_kernel<D, CAP, BIAS>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM);
  if (e != cudaSuccess) return (int)e;
  launch_early(0, k, grid, kThreads, Cfg<D>::SMEM, stream, tq, to, td, a);
  return (int)cudaGetLastError();
}

// dK and dV of a token = the shares' sums, added in order and rounded once.
__global__ void join_parts_kernel(const float* __restrict__ partial, int parts, long stride, long tokens, int width,
                                  __nv_bfloat16* __restrict__ dqkv, long ld, long col0) {
  pdl_trigger();
  pdl_wait();
  const long n = tokens * (width / 8);
  for (long u = blockIdx.x * (long)blockDim.x + threadIdx.x; u < n; u += (long)gridDim.x * blockDim.x) {
    const long tok = u / (width / 8);
    const int c = (int)(u - tok * (width / 8)) * 8;
    const float* p = partial + tok * width + c;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
    for (int k = 0; k < parts; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(p + k * stride), w = *reinterpret_cast<const float4*>(p + k * stride + 4);
      x = make_float4(x.x + v.x, x.y + v.y, x.z + v.z, x.w + v.w);
      y = make_float4(y.x + w.x, y.y + w.y, y.z + w.z, y.w + w.w);
    }
    *reinterpret_cast<uint4*>(dqkv + tok * ld + col0 + c) =
        make_uint4(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w), pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
  }
}

}  // namespace dkv
}  // namespace mattn

// Few key tiles and shared heads: an item is a share of the K/V head's query heads, so that every SM gets work
// (two items each at least, which leaves the heaviest-first order something to balance); the shares' 32-bit sums are
// joined afterwards.  One K/V head of 128 key tiles (S = 16384, 4 query heads) took 551 us as 128 items and
// 247 us with the join as 512.
//
// Waits for the end of an item give up after 2 s.  A (query head, query tile) pair takes 1.2 us (d = 64) to 3.4 us (d = 128,
// scores beyond the cap, distance bias), in loops of seconds under the power limit, so an item of kAttnMaxTiles of them ends
// within 0.9 s; longer ones are split too.
int masked_attn_dkv_parts(int B, int S, int nh, int nkv, int num_sms) {
  const long items = (long)B * nkv * ((S + mattn::BT - 1) / mattn::BT);
  const int group = nh / nkv;
  const long n_t = (S + mattn::BT - 1) / mattn::BT;
  for (int p = 1; p < group; ++p)
    if (group % p == 0 && items * p >= 2L * num_sms && group / p * n_t <= kAttnMaxTiles) return p;
  return group;
}

int masked_attn_dkv(const AttnCall& c, const void* dout, long do_ss, long do_sb, const float* ld, float* partial,
                    int parts, void* dqkv, int* err, int num_sms, cudaStream_t stream) {
  using namespace mattn;
  const int n_t = (c.S + BT - 1) / BT;
  const long items = (long)c.B * c.nkv * n_t * parts;
  if (parts < 1 || (c.nh / c.nkv) % parts || (parts > 1 && !partial)) return -3;
  if (items > INT_MAX / 2) return -1;
  CUtensorMap tq, to, td;
  int rc = make_tmap_bf16_3d(&tq, c.qkv, c.B, c.S, (long)(c.nh + 2 * c.nkv) * c.d, c.qkv_ss, c.qkv_sb, 64, BT);
  if (rc) return rc - 10;
  rc = make_tmap_bf16_3d(&to, dout, c.B, c.S, (long)c.nh * c.d, do_ss, do_sb, 64, BT);
  if (rc) return rc - 20;
  const long width = (long)(c.nh + 2 * c.nkv) * c.d;
  rc = make_tmap_bf16_3d(&td, dqkv, c.B, c.S, width, width, width * c.S, 64, BT);
  if (rc) return rc - 30;
  dkv::Args a;
  a.B = c.B;
  a.S = c.S;
  a.nh = c.nh;
  a.nkv = c.nkv;
  a.n_t = n_t;
  a.parts = parts;
  a.heads = c.nh / c.nkv / parts;
  a.by_parts = FastDiv(parts);
  a.by_nkv = FastDiv(c.nkv);
  a.by_B = FastDiv(c.B);
  a.by_tiles = FastDiv(n_t);
  a.partial = partial;
  a.mask = Mask{c.rows, static_cast<const int4*>(c.qstat), static_cast<const int4*>(c.kstat), c.order_k};
  a.slopes = c.slopes;
  a.score = score_constants(c.scale, c.cap);
  a.scale = c.scale;
  a.ld = ld;
  a.dqkv = static_cast<__nv_bfloat16*>(dqkv);
  a.err = err;
  const int grid = (int)std::max(1L, std::min(items, (long)num_sms));
  const bool cap = c.cap > 0.f, bias = c.slopes != nullptr;
  if (c.d == 64) {
    if (cap) rc = bias ? dkv::launch<64, true, true>(tq, to, td, a, grid, stream) : dkv::launch<64, true, false>(tq, to, td, a, grid, stream);
    else rc = bias ? dkv::launch<64, false, true>(tq, to, td, a, grid, stream) : dkv::launch<64, false, false>(tq, to, td, a, grid, stream);
  } else if (c.d == 128) {
    if (cap) rc = bias ? dkv::launch<128, true, true>(tq, to, td, a, grid, stream) : dkv::launch<128, true, false>(tq, to, td, a, grid, stream);
    else rc = bias ? dkv::launch<128, false, true>(tq, to, td, a, grid, stream) : dkv::launch<128, false, false>(tq, to, td, a, grid, stream);
  } else {
    rc = -2;
  }
  if (rc || parts == 1) return rc;
  const long tokens = (long)c.B * c.S, wid = 2L * c.nkv * c.d;
  const long units = tokens * (wid / 8);
  launch_early(0, dkv::join_parts_kernel, (unsigned)std::min((units + 255) / 256, 8L * num_sms), 256, 0, stream, partial, parts,
           tokens * wid, tokens, (int)wid, static_cast<__nv_bfloat16*>(dqkv), width, (long)c.nh * c.d);
  return (int)cudaGetLastError();
}

}  // namespace mmb
