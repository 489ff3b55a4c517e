// Masked attention forward for sm_100a: document and prefix masks, scores capped
// by a tanh, a bias linear in the distance, shared K/V heads, any sequence length.
//
//   O_i = sum_j softmax_j(x_ij) v_j,  LSE_i = log sum_j exp(x_ij)   (x: masked_attn.cuh)
//
// A row that sees nothing gives O = 0 and LSE = -inf.  The running maximum, the
// row sum and O stay in 32 bits; P is rounded to bf16 once, as the operand of
// P V, relative to a maximum at most 2^8 stale.
//
// Persistent grid, one CTA per SM.  A work item is (batch, head, two adjacent
// 128-row query tiles); both tiles share the K/V tiles they both need, so a
// K/V tile is fetched once per 256 queries.  Only the key tiles that a query tile's
// rows can see are visited, and only those that some row does not see completely
// pay for a mask.  Roles (16 warps):
//
//   warp 0       TMA: Q tiles per item; K_j / V_j into an NS-stage ring
//   warps 1, 2   one thread each issues S_i = Q_i K_j^T and O_i += P_i V_j of its tile (warp 1 also
//                allocates TMEM); with one thread for both, the tile that is ready waited for the
//                other one's P: 77 us instead of 67 at 16 x 1024 tokens, 12 heads of 64
//   warp 3       decodes work items and hands them out through a ring
//   warps 4-7,   softmax of tile 0 / tile 1, a thread per query row: scores out of
//   warps 8-11   TMEM, transform, mask, running maximum, P back into TMEM as bf16
//   warps 12-15  epilogue of both tiles: O / row sum -> bf16, LSE; it runs while the
//                softmax warps are in the next item
//
// O is rescaled in TMEM only when a row's maximum grew by more than 2^8; until then
// P, O and the row sum share the stale maximum, so nothing is approximated.
//
// d = 64: P has its own TMEM columns and Q two buffers, so S_i(j+1) is computed while
// P_i(j) is.  d = 128: S and O of two tiles fill TMEM, P overwrites S, and the two tiles
// alternate between the tensor core and the softmax.
//
// What bounds it, causal rows: at d = 64 the exponentials (16 a cycle and SM), which the chain score - maximum -
// exponential - P leaves idle in part: 16384 tokens, 4 heads: 200 us, 62 % of their rate; 16 x 1024 tokens, 12 heads:
// 62 us, 42 %, with five steps an item.  d = 128: tensor cores and exponentials alike; 16384 tokens, 8 heads: 436 us,
// 1270 TFLOP/s over the tiles visited.
//
// Every wait is bounded; on a time-out the kernel records an error code, all roles wind
// down, loads and MMAs in flight are waited for (bounded), TMEM is freed and the CTA returns.
#include "masked_attn.cuh"

namespace mmb {
namespace mattn {
namespace fwd {

constexpr int kThreads = 512;
constexpr float kRescaleLog2 = 8.0f;

template <int D>
struct Cfg {
  static constexpr int TILE = BT * D * 2;
  static constexpr int NS = (D == 64) ? 4 : 2;  // K/V ring stages
  static constexpr bool SEP = (D == 64);        // P in its own TMEM columns
  static constexpr int QB = SEP ? 2 : 1;
  static constexpr int Q_OFF = 0;  // [QB][Q0, Q1]
  static constexpr int K_OFF = QB * 2 * TILE;
  static constexpr int V_OFF = K_OFF + NS * TILE;
  static constexpr int ML_OFF = V_OFF + NS * TILE;  // [2][128] (maximum, row sum)
  static constexpr int OUT_OFF = ML_OFF + 2 * BT * 8;  // 4 epilogue warps x 32 rows x 64 columns bf16
  static constexpr int ITEM_OFF = OUT_OFF + 4 * 4096;  // [kRing] work items
  static constexpr int BAR_OFF = ITEM_OFF + kRing * 64;
  static constexpr int SMEM = 1024 + BAR_OFF + 512;
  // Registers: 128 a thread at launch, 65536 in all.  d = 128: an epilogue that reads O 16 columns at a time leaves the
  // softmax 200 and with them fewer spills (4 x 2048 x 16 causal 74.8 us instead of 77.4, capped 121 instead of 127); at
  // d = 64 the same split was slower (S = 16384: 240 us instead of 200).
  static constexpr int SOFTMAX_REGS = D == 128 ? 200 : 192, EPI_REGS = D == 128 ? 56 : 72, EPI_COLS = D == 128 ? 16 : 32;
  static constexpr uint32_t T_S0 = 0, T_S1 = 128, T_O0 = 256, T_O1 = 256 + D;
  static constexpr uint32_t T_P0 = SEP ? 384 : T_S0, T_P1 = SEP ? 448 : T_S1;
};

struct Args {
  int B, S, nh, nkv, n_t, n_pairs;
  FastDiv by_nh, by_B, by_pairs, by_group;
  Mask mask;
  const float* slopes;  // [nh] or nullptr
  Score score;
  float* lse;  // [B, nh, S] natural log
  __nv_bfloat16* out;   // [B, S, nh * D]
  int* err;
};

struct alignas(16) Item {
  int b, h, t0, t1;  // b < 0: no more items; t0 < 0: only tile t1 (odd number of tiles)
  int2 r0, r1;       // key tiles of t0, t1
  int2 f0, f1;       // those of them that need no mask
  int lo, hi;        // union of the key tiles
};
static_assert(sizeof(Item) <= 64, "ring entry");
constexpr int kConsumers = 1 + 2 + 8 + 4;  // TMA and MMA threads, softmax and epilogue warps

__device__ __forceinline__ Item decode(const Args& a, int item) {
  const int li = a.by_nh.quot(item);
  Item it;
  it.h = item - li * a.nh;
  int p;
  if (a.mask.order) {
    const int e = ordered(a.mask.order, li, a.B * a.n_pairs);
    it.b = a.by_pairs.quot(e);
    p = e - it.b * a.n_pairs;
  } else {  // causal rows: the longest first
    const int q = a.by_B.quot(li);
    it.b = li - q * a.B;
    p = a.n_pairs - 1 - q;
  }
  it.t1 = (a.n_t & 1) ? 2 * p : 2 * p + 1;
  it.t0 = it.t1 - 1;
  it.r0 = it.f0 = make_int2(0, 0);
  if (it.t0 >= 0) {
    key_tiles(a.mask, it.b, a.n_t, it.t0, it.r0, it.f0);
  }
  key_tiles(a.mask, it.b, a.n_t, it.t1, it.r1, it.f1);
  const bool a0 = it.r0.y > it.r0.x, a1 = it.r1.y > it.r1.x;
  it.lo = a0 ? (a1 ? min(it.r0.x, it.r1.x) : it.r0.x) : it.r1.x;
  it.hi = max(it.r0.y, it.r1.y);
  if (!a0 && !a1) it.hi = it.lo;
  return it;
}

// Whether the exponentials of the two tiles take turns.
template <int D>
constexpr bool kTurns = D == 128;

constexpr int kIssueRegs = 56;
static_assert(4 * kIssueRegs + 8 * Cfg<64>::SOFTMAX_REGS + 4 * Cfg<64>::EPI_REGS <= 16 * 128 &&
                  4 * kIssueRegs + 8 * Cfg<128>::SOFTMAX_REGS + 4 * Cfg<128>::EPI_REGS <= 16 * 128,
              "registers of the launch");

template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
    masked_attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_out,
                           const Args a) {
  pdl_trigger();
  using C = Cfg<D>;
  constexpr int NS = C::NS;
  constexpr int QB = C::QB;
  constexpr bool SEP = C::SEP;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sQ = smem + C::Q_OFF;
  uint8_t* sK = smem + C::K_OFF;
  uint8_t* sV = smem + C::V_OFF;
  float2* sML = reinterpret_cast<float2*>(smem + C::ML_OFF);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* q_full = bars;            // [2]
  uint64_t* q_empty = bars + 2;       // [2]
  uint64_t* k_full = bars + 4;        // [NS]
  uint64_t* k_empty = k_full + NS;    // [NS]
  uint64_t* v_full = k_empty + NS;    // [NS]
  uint64_t* v_empty = v_full + NS;    // [NS]
  uint64_t* s_full = v_empty + NS;    // [2]  S_i computed
  uint64_t* s_free = s_full + 2;      // [2]  S_i in registers (SEP; 4 warps)
  uint64_t* p_full = s_free + 2;      // [2][2]  first / other 64 keys of P_i written (4 warps)
  uint64_t* p_free = p_full + 4;      // [2]  PV_i that read P_i complete (SEP)
  uint64_t* o_full = p_free + 2;      // [2]  last PV_i of the item complete
  uint64_t* o_free = o_full + 2;      // [2]  O_i and its statistics read by the epilogue (4 warps)
  uint64_t* ml_full = o_free + 2;     // [2]  statistics of the item written (4 warps)
  uint64_t* turn = ml_full + 2;       // [2][4]  exponentials of a joint step issued, per tile and sub-partition
  uint64_t* ring_full = turn + 8;     // [kRing]
  uint64_t* ring_empty = ring_full + kRing;  // [kRing]
  uint64_t* drain = ring_empty + kRing;      // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Ring<Item> ring{reinterpret_cast<Item*>(smem + C::ITEM_OFF), ring_full, ring_empty};

  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) mbar_init(&turn[i], 1);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&ring_full[i], 1);
      mbar_init(&ring_empty[i], kConsumers);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 2);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&p_free[i], 1);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_free[i], 4);
      mbar_init(&ml_full[i], 4);
      mbar_init(&drain[i], 1);
    }
    for (int s = 0; s < NS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 2);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 2);
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tm_qkv);
    prefetch_tmap(&tm_out);
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
    reg_dec<kIssueRegs>();
    if (warp == 0 && elect_one()) {
      // ---------------------------------------------------------------- TMA
      int kv = 0, it = 0, q_issued = -1;
      bool ok = true;
      Item w;
      for (int k = 0; (ok = ring.get_thread(w, k, a.err, abort_flag)) && w.b >= 0; ++k) {
        if (w.lo >= w.hi) continue;
        const bool a0 = w.r0.y > w.r0.x, a1 = w.r1.y > w.r1.x;
        const int hk = a.by_group.quot(w.h);
        const int qx = w.h * D, kx = (a.nh + hk) * D, vx = (a.nh + a.nkv + hk) * D;
        const int qb = it % QB;
        if (it >= QB && !bwait(&q_empty[qb], ((it / QB) - 1) & 1, a.err, abort_flag)) { ok = false; break; }
        uint8_t* qd = sQ + qb * 2 * C::TILE;
        mbar_expect_tx(&q_full[qb], ((a0 ? 1 : 0) + (a1 ? 1 : 0)) * C::TILE);
        if (a0) load_tile<D>(qd, &tm_qkv, &q_full[qb], qx, w.t0 * BT, w.b);
        if (a1) load_tile<D>(qd + C::TILE, &tm_qkv, &q_full[qb], qx, w.t1 * BT, w.b);
        q_issued = it;
        for (int j = w.lo; j < w.hi; ++j, ++kv) {
          const int s = kv % NS, n = kv / NS;
          if (n > 0 && !bwait(&k_empty[s], (n - 1) & 1, a.err, abort_flag)) { ok = false; break; }
          mbar_expect_tx(&k_full[s], C::TILE);
          load_tile<D>(sK + s * C::TILE, &tm_qkv, &k_full[s], kx, j * BT, w.b);
          if (n > 0 && !bwait(&v_empty[s], (n - 1) & 1, a.err, abort_flag)) {
            ++kv;  // the K load of this slot is in flight
            ok = false;
            break;
          }
          mbar_expect_tx(&v_full[s], C::TILE);
          load_tile<D>(sV + s * C::TILE, &tm_qkv, &v_full[s], vx, j * BT, w.b);
        }
        if (!ok) break;
        ++it;
      }
      if (!ok) {
        // let the loads in flight land before the CTA's shared memory goes away
        for (int u = max(0, q_issued - QB + 1); u <= q_issued; ++u) drain_wait(&q_full[u % QB], (u / QB) & 1);
        for (int u = max(0, kv - NS); u < kv; ++u) {
          drain_wait(&k_full[u % NS], (u / NS) & 1);
          drain_wait(&v_full[u % NS], (u / NS) & 1);
        }
      }
    } else if ((warp == 1 || warp == 2) && elect_one()) {
      // ---------------------------------------------------------------- MMA, tile grp of every item
      const int grp = warp - 1;
      const uint32_t t_s = tmem + (grp == 0 ? C::T_S0 : C::T_S1);
      const uint32_t t_p = tmem + (grp == 0 ? C::T_P0 : C::T_P1);
      const uint32_t t_o = tmem + (grp == 0 ? C::T_O0 : C::T_O1);
      int kv = 0, it = 0;
      int sc = 0, pc = 0, ic = 0;  // S issued (s_free phases), P consumed (p_full), items with keys (o_free)
      bool ok = true;
      uint32_t q_addr = 0;
      // S of the K stage of loop position u; the stage, and after an item's last one Q, are released either way
      auto issue_s = [&](int u, bool on, bool last) -> bool {
        const int st = u % NS;
        if (!bwait(&k_full[st], (u / NS) & 1, a.err, abort_flag)) return false;
        if (on) {
          if (SEP && sc > 0 && !bwait(&s_free[grp], (sc - 1) & 1, a.err, abort_flag)) return false;
          ++sc;
          tc_fence_after();
          mma_abt<D>(t_s, q_addr, smem_u32(sK + st * C::TILE));
          umma_commit(&s_full[grp]);
        }
        umma_commit(&k_empty[st]);
        if (last) umma_commit(&q_empty[it % QB]);
        return true;
      };
      auto issue_pv = [&](int u, bool on, bool first, bool last) -> bool {
        const int st = u % NS;
        if (!bwait(&v_full[st], (u / NS) & 1, a.err, abort_flag)) return false;
        if (on) {
          // the first 64 keys' share runs while the softmax is at the other 64
          if (!bwait(&p_full[2 * grp], pc & 1, a.err, abort_flag)) return false;
          if (first && ic > 0 && !bwait(&o_free[grp], (ic - 1) & 1, a.err, abort_flag)) return false;
          tc_fence_after();
          mma_tmem_b<D, 64, 32, 0, 4>(t_o, t_p, smem_u32(sV + st * C::TILE), !first);
          if (!bwait(&p_full[2 * grp + 1], pc & 1, a.err, abort_flag)) return false;
          ++pc;
          tc_fence_after();
          mma_tmem_b<D, 64, 32, 4, 8>(t_o, t_p, smem_u32(sV + st * C::TILE), true);
          if (SEP) umma_commit(&p_free[grp]);
          if (last) umma_commit(&o_full[grp]);
        }
        umma_commit(&v_empty[st]);
        return true;
      };
      Item w;
      for (int k = 0; (ok = ring.get_thread(w, k, a.err, abort_flag)) && w.b >= 0; ++k) {
        if (w.lo >= w.hi) continue;
        const int2 range = grp == 0 ? w.r0 : w.r1;
        const int qb = it % QB;
        q_addr = smem_u32(sQ + (qb * 2 + grp) * C::TILE);
        if (!bwait(&q_full[qb], (it / QB) & 1, a.err, abort_flag)) { ok = false; break; }
        auto on = [&](int j) { return j >= range.x && j < range.y; };
        if (!issue_s(kv, on(w.lo), w.lo + 1 == w.hi)) { ok = false; break; }
        for (int j = w.lo; j < w.hi; ++j, ++kv) {
          // d = 64: the next scores first, they only need the softmax to have read the current ones;
          // d = 128: P overwrites S, the next scores follow P V
          if (SEP && j + 1 < w.hi && !issue_s(kv + 1, on(j + 1), j + 2 == w.hi)) { ok = false; break; }
          if (!issue_pv(kv, on(j), j == range.x, j == range.y - 1)) { ok = false; break; }
          if (!SEP && j + 1 < w.hi && !issue_s(kv + 1, on(j + 1), j + 2 == w.hi)) { ok = false; break; }
        }
        if (!ok) break;
        ++it;
        if (range.x < range.y) ++ic;
      }
      if (!ok) {
        umma_commit(&drain[grp]);
        drain_wait(&drain[grp], 0);
      }
    } else if (warp == 3 && elect_one()) {
      // ---------------------------------------------------------------- work items
      const int n_items = a.B * a.nh * a.n_pairs;
      Item w;
      for (int r = 0, item;; ++r) {
        item = snake_item(r);
        if (item < n_items) w = decode(a, item);
        else w.b = -1;
        if (!ring.put(w, r, a.err, abort_flag) || w.b < 0) break;
      }
    }
    __syncwarp();
  } else if (warp < 12) {
    // ------------------------------------------------------------------ softmax
    reg_inc<C::SOFTMAX_REGS>();
    const int grp = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;  // query row within the tile (TMEM lane)
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + (grp == 0 ? C::T_S0 : C::T_S1) + lane_off;
    const uint32_t t_p = tmem + (grp == 0 ? C::T_P0 : C::T_P1) + lane_off;
    const uint32_t t_o = tmem + (grp == 0 ? C::T_O0 : C::T_O1) + lane_off;
    const Score k = a.score;
    int sc = 0, pc = 0, ic = 0, nj = 0;  // nj: steps that both tiles take
    bool ok = true;
    Item w;
    for (int n = 0; (ok = ring.get_warp(w, n, a.err, abort_flag)) && w.b >= 0; ++n) {
      const int t = grp == 0 ? w.t0 : w.t1;
      const int2 range = grp == 0 ? w.r0 : w.r1, other = grp == 0 ? w.r1 : w.r0, full = grp == 0 ? w.f0 : w.f1;
      if (range.x >= range.y) continue;
      const int i = t * BT + row;
      int start = 0, end = i + 1;
      if (a.mask.rows) {
        const int* tr = a.mask.rows + ((size_t)w.b * a.n_t + t) * (4 * BT) + row;
        start = tr[0];
        end = tr[BT];
      }
      float slope = 0.f;
      if (BIAS) slope = a.slopes[w.h] * kLog2e;
      float m = -INFINITY, l = 0.f;
      for (int j = range.x; j < range.y; ++j) {
        if (!wwait(&s_full[grp], sc & 1, a.err, abort_flag)) { ok = false; break; }
        ++sc;
        tc_fence_after();
        uint32_t s[128];
        tmem_ld_32x32b_x32(t_s + 0, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
        tmem_ld_32x32b_x32(t_s + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
        tmem_ld_32x32b_x32(t_s + 64, *reinterpret_cast<uint32_t(*)[32]>(&s[64]));
        tmem_ld_32x32b_x32(t_s + 96, *reinterpret_cast<uint32_t(*)[32]>(&s[96]));
        tmem_wait_ld();
        if (SEP) warp_arrive(&s_free[grp]);  // the next S_i may be computed into these columns
        if (CAP) cap_in_place(s, k);
        if (CAP || BIAS) {
          const float dist = (float)(j * BT - i);
#pragma unroll
          for (int c = 0; c < 128; c += 2) {
            float2 x = mul2(pair(s[c], s[c + 1]), pair(CAP ? k.cap : k.mul));
            if (BIAS) {
              x.x = fmaf(-slope, fabsf(dist + (float)c), x.x);
              x.y = fmaf(-slope, fabsf(dist + (float)(c + 1)), x.y);
            }
            s[c] = __float_as_uint(x.x);
            s[c + 1] = __float_as_uint(x.y);
          }
        }
        if (j < full.x || j >= full.y) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const uint32_t seen = seen_bits(start, end, j * BT + 32 * g);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen & (1u << e))) s[32 * g + e] = 0xff800000u;  // -inf
          }
        }
        float mx[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) mx[u] = __uint_as_float(s[u]);
#pragma unroll
        for (int c = 8; c < 120; c += 16) {
#pragma unroll
          for (int u = 0; u < 8; ++u)
            mx[u] = max3(mx[u], __uint_as_float(s[c + 2 * u]), __uint_as_float(s[c + 2 * u + 1]));
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) mx[u] = fmaxf(mx[u], __uint_as_float(s[120 + u]));
        float mt = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7]));
        if (!CAP && !BIAS) mt *= k.mul;
        const bool need = mt > m + kRescaleLog2;
        const bool any_need = __any_sync(0xffffffffu, need) != 0;
        float alpha = 1.f;
        if (need) {
          alpha = fast_exp2(m - mt);  // m = -inf (nothing seen yet): 0
          m = mt;
        }
        const float mu = m == -INFINITY ? 0.f : m;  // a row that has seen nothing: every exponential is 0
        // SEP: before P_i's columns (and O_i) are written, the PV that read the previous P_i (and last wrote O_i) must be
        // complete.  With a cap that wait sits behind the first half of the exponentials unless O_i has to be rescaled
        // (16 x 1024 tokens, 12 heads of 64: 112 us instead of 123); without one it comes first: the two tiles then fall into step less
        // (S = 16384: 206 us instead of 225).
        bool waited = !SEP || pc == 0;
        if (!waited && (!CAP || (any_need && j > range.x))) {
          if (!wwait(&p_free[grp], (pc - 1) & 1, a.err, abort_flag)) { ok = false; break; }
          tc_fence_after();
          waited = true;
        }
        if (any_need && j > range.x) {
          // d = 128: PV_i(j-1) was issued before S_i(j), which is complete
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(t_o + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st_x32(t_o + c * 32, o);
          }
        }
        // the exponentials of the two tiles take turns, one warp of each on every SM sub-partition: while one
        // fills the pipes the other waits for its scores, takes its maximum and stores its P
        const bool joint = kTurns<D> && j >= other.x && j < other.y;
        if (joint && (grp == 1 || nj > 0)) {
          if (!wwait(&turn[(grp ^ 1) * 4 + (warp & 3)], (grp == 1 ? nj : nj - 1) & 1, a.err, abort_flag)) {
            ok = false;
            break;
          }
        }
        float2 rs[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) rs[u] = pair(0.f);
#pragma unroll
        for (int hcol = 0; hcol < 2; ++hcol) {
          uint32_t pk[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int c = hcol * 64 + 2 * e;
            float2 x = pair(s[c], s[c + 1]);
            x = (CAP || BIAS) ? add2(x, pair(-mu)) : fma2(x, pair(k.mul), pair(-mu));
            x = exp2_pair(x);
            rs[e & 3] = add2(rs[e & 3], x);
            pk[e] = pack_bf16x2(x.x, x.y);
          }
          if (!waited) {
            if (!wwait(&p_free[grp], (pc - 1) & 1, a.err, abort_flag)) { ok = false; break; }
            tc_fence_after();
            waited = true;
          }
          tmem_st_x32(t_p + hcol * 32, pk);
          tmem_wait_st();
          warp_arrive(&p_full[2 * grp + hcol]);
        }
        if (!ok) break;
        ++pc;
        if (joint) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&turn[grp * 4 + (warp & 3)]);
          ++nj;
        }
        rs[0] = add2(add2(rs[0], rs[1]), add2(rs[2], rs[3]));
        l = l * alpha + (rs[0].x + rs[0].y);
      }
      if (!ok) break;
      // hand the statistics to the epilogue
      if (ic > 0 && !wwait(&o_free[grp], (ic - 1) & 1, a.err, abort_flag)) { ok = false; break; }
      ++ic;
      sML[grp * BT + row] = make_float2(m, l);
      warp_arrive(&ml_full[grp]);
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    reg_dec<C::EPI_REGS>();
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    uint8_t* stg = smem + C::OUT_OFF + (warp & 3) * 4096;
    int ic[2] = {0, 0};
    bool ok = true;
    Item w;
    for (int n = 0; ok && (ok = ring.get_warp(w, n, a.err, abort_flag)) && w.b >= 0; ++n) {
#pragma unroll
      for (int grp = 0; grp < 2; ++grp) {
        const int t = grp == 0 ? w.t0 : w.t1;
        if (t < 0) continue;
        const int2 range = grp == 0 ? w.r0 : w.r1;
        const int i = t * BT + row;
        const bool in = i < a.S;
        __nv_bfloat16* orow = a.out + ((size_t)w.b * a.S + i) * ((size_t)a.nh * D) + (size_t)w.h * D;
        float* lse = a.lse + ((size_t)w.b * a.nh + w.h) * a.S + i;
        if (range.x >= range.y) {  // no row of the tile sees anything
          if (in) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) store_zero<32>(orow + c * 32);
            *lse = -INFINITY;
          }
          continue;
        }
        if (!wwait(&ml_full[grp], ic[grp] & 1, a.err, abort_flag) ||
            !wwait(&o_full[grp], ic[grp] & 1, a.err, abort_flag)) {
          ok = false;
          break;
        }
        ++ic[grp];
        tc_fence_after();
        const float2 ml = sML[grp * BT + row];
        const bool seen = ml.y != 0.f;
        const float inv = seen ? 1.f / ml.y : 0.f;
        const uint32_t t_o = tmem + (grp == 0 ? C::T_O0 : C::T_O1) + lane_off;
#pragma unroll
        for (int c = 0; c < D; c += C::EPI_COLS) {
          uint32_t o[C::EPI_COLS];
          tmem_ld(t_o + c, o);
          if (c % 64 == 0 && lane == 0) bulk_wait_read<0>();  // the last store has read the staged rows
          tmem_wait_ld();
          __syncwarp();
          if (c == D - C::EPI_COLS) warp_arrive(&o_free[grp]);  // O and the statistics are in registers
          stage_row(stg, 0, lane, c % 64, o, inv);
          if ((c + C::EPI_COLS) % 64 == 0) {
            fence_proxy_async_smem();
            __syncwarp();
            const int row0 = t * BT + (warp & 3) * 32;
            if (lane == 0 && row0 < a.S) {
              tma_store_3d(&tm_out, stg, w.h * D + (c / 64) * 64, row0, w.b);
              bulk_commit();
            }
          }
        }
        if (in) *lse = seen ? ml.x * kLn2 + logf(ml.y) : -INFINITY;
      }
    }
    if (lane == 0) bulk_wait<0>();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool CAP, bool BIAS>
int launch(const CUtensorMap& tm, const CUtensorMap& to, const Args& a, int grid, cudaStream_t stream) {
  auto k = masked_attn_fwd_kernel<D, CAP, BIAS>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM);
  if (e != cudaSuccess) return (int)e;
  launch_early(0, k, grid, kThreads, Cfg<D>::SMEM, stream, tm, to, a);
  return (int)cudaGetLastError();
}

}  // namespace fwd
}  // namespace mattn

int masked_attn_fwd(const AttnCall& c, void* out, float* lse, int* err, int num_sms, cudaStream_t stream) {
  using namespace mattn;
  const int n_t = (c.S + BT - 1) / BT;
  const long items = (long)c.B * c.nh * ((n_t + 1) / 2);
  if (items > INT_MAX / 2) return -1;
  CUtensorMap tm, to;
  int rc = make_tmap_bf16_3d(&tm, c.qkv, c.B, c.S, (long)(c.nh + 2 * c.nkv) * c.d, c.qkv_ss, c.qkv_sb, 64, BT);
  if (rc) return rc - 10;
  rc = make_tmap_bf16_3d(&to, out, c.B, c.S, (long)c.nh * c.d, (long)c.nh * c.d, (long)c.S * c.nh * c.d, 64, 32);
  if (rc) return rc - 20;
  fwd::Args a;
  a.B = c.B;
  a.S = c.S;
  a.nh = c.nh;
  a.nkv = c.nkv;
  a.n_t = n_t;
  a.n_pairs = (n_t + 1) / 2;
  a.by_nh = FastDiv(c.nh);
  a.by_B = FastDiv(c.B);
  a.by_pairs = FastDiv(a.n_pairs);
  a.by_group = FastDiv(c.nh / c.nkv);
  a.mask = Mask{c.rows, static_cast<const int4*>(c.qstat), static_cast<const int4*>(c.kstat), c.order_p};
  a.slopes = c.slopes;
  a.score = score_constants(c.scale, c.cap);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.lse = lse;
  a.err = err;
  const int grid = (int)std::max(1L, std::min(items, (long)num_sms));
  const bool cap = c.cap > 0.f, bias = c.slopes != nullptr;
  if (c.d == 64) {
    if (cap) return bias ? fwd::launch<64, true, true>(tm, to, a, grid, stream) : fwd::launch<64, true, false>(tm, to, a, grid, stream);
    return bias ? fwd::launch<64, false, true>(tm, to, a, grid, stream) : fwd::launch<64, false, false>(tm, to, a, grid, stream);
  }
  if (c.d == 128) {
    if (cap) return bias ? fwd::launch<128, true, true>(tm, to, a, grid, stream) : fwd::launch<128, true, false>(tm, to, a, grid, stream);
    return bias ? fwd::launch<128, false, true>(tm, to, a, grid, stream) : fwd::launch<128, false, false>(tm, to, a, grid, stream);
  }
  return -2;
}

}  // namespace mmb
