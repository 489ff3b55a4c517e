// Masked attention backward, query side: dQ, and the row statistics of the key side.
//
//   P_ij = exp(x_ij - LSE_i),  Delta_i = sum_c dO_ic O_ic
//   dS_ij = P_ij (dO_i.v_j - Delta_i) (1 - tanh^2 u_ij),  dQ_i = s sum_j dS_ij k_j
//
// The backward is two passes over the visible tiles, one that stays with a query
// tile (this file) and one that stays with a key tile (masked_attn_dkv.cu).  Scores
// are computed twice, but each gradient is summed in one place in one order, in
// 32-bit TMEM accumulators: no atomics, no zeroed 32-bit copy of dQ, no conversion
// pass, and the same inputs give the same bits.  dS is rounded to bf16 once, as
// the operand of its products.
//
// row_stats_kernel: one pass over ctx and dO computes Delta and stores it with LSE, both negated and in the units of
// the softmax, in an array padded to whole tiles, from which both passes fetch a tile's rows with bulk copies.
// (Two warps of the query-side kernel computing it for the item ahead kept pace only with batches of loads
// that took the registers of the softmax warps; as a kernel of its own it is bound by reading ctx and dO.)
//
// masked_attn_dq_kernel: persistent grid, one CTA per SM; a work item is (batch, head, 128-row query tile).
// Roles (20 warps):
//
//   warp 0      TMA: Q, dO and row statistics per item; K_j and V_j into rings
//   warp 1      TMEM allocation; one thread issues S = Q K_j^T (two TMEM buffers), dP = dO V_j^T
//               and dQ += dS K_j (dS read from TMEM): S of the next tile before dS of this one is
//               ready, dP of the next as soon as this one has been read
//   warp 2      hands out the work items
//   warp 3      stores finished dQ tiles from the K stage they were staged in
//   warps 4-19  dS: four warps share 32 query rows, each has 32 of the 128 keys
//
// dS overwrites the S columns it came from: every warp's 32 keys start 32 columns apart.
// A warp's step is a chain of waits, a TMEM load, exponentials, another wait and load and the
// store; four warps on each SM sub-partition fill one another's gaps (with two, 64 keys each, 16 x 1024
// tokens of 12 heads of 64 took 86 us instead of 83).
//
// dQ of an item stays in TMEM until the next item's first tile: its last product runs while that tile's P is
// computed, and a warp of its own stores it (68 us before, 58 with it at the same size).
//
// What bounds it, causal rows: at d = 64 the chain of a tile (128 x 128 scores between two products, with 16384
// exponentials at 16 a cycle in it), at d = 128 the tensor cores.  16 x 1024 tokens, 12 heads of 64: 58 us, 750 TFLOP/s
// over the tiles visited; 16384 tokens, 8 heads of 128: 572 us, 1450 TFLOP/s.
#include "masked_attn.cuh"

namespace mmb {
namespace mattn {
namespace dq {

constexpr int kThreads = 640;
constexpr int kWarps = 16;  // of the softmax gradient

template <int D>
struct Cfg {
  static constexpr int TILE = BT * D * 2;
  static constexpr int QB = (D == 64) ? 2 : 1;  // Q / dO buffers
  static constexpr int NK = (D == 64) ? 4 : 3;  // K ring: held from S(j) to dQ(j), one tile longer than V
  static constexpr int NV = (D == 64) ? 4 : 2;
  static constexpr int Q_OFF = 0;               // [QB][Q, dO]
  static constexpr int K_OFF = QB * 2 * TILE;
  static constexpr int V_OFF = K_OFF + NK * TILE;
  static constexpr int ST_OFF = V_OFF + NV * TILE;  // [QB][-LSE log2 e 128, -Delta 128]
  static constexpr int ITEM_OFF = ST_OFF + QB * BT * 8;  // [kRing] work items
  static constexpr int BAR_OFF = ITEM_OFF + kRing * 32;
  static constexpr int SMEM = 1024 + BAR_OFF + 352;
  static constexpr uint32_t T_S = 0, T_DP = 256, T_DQ = 384;  // S: two buffers of 128 columns
};
static_assert(Cfg<128>::SMEM <= 227 * 1024 && Cfg<64>::SMEM <= 227 * 1024, "shared memory of one CTA");

struct Args {
  int B, S, nh, nkv, n_t;
  FastDiv by_nh, by_B, by_tiles, by_group;
  Mask mask;
  const float* slopes;
  Score score;
  float scale;
  const float* ld;            // [B, nh, n_t, 2, 128] -LSE log2 e (-inf: the row takes no part), -Delta
  __nv_bfloat16* dqkv;        // [B, S, (nh + 2 nkv) * D]
  int* err;
};

struct alignas(16) Item {
  int b, h, t;  // b < 0: no more items
  int2 r, f;    // key tiles, and those of them that need no mask
};
static_assert(sizeof(Item) <= 32, "ring entry");
constexpr int kConsumers = 1 + 1 + 1 + kWarps;  // TMA and MMA threads, store and softmax warps

__device__ __forceinline__ Item decode(const Args& a, int item) {
  const int li = a.by_nh.quot(item);
  Item it;
  it.h = item - li * a.nh;
  if (a.mask.order) {
    const int e = ordered(a.mask.order, li, a.B * a.n_t);
    it.b = a.by_tiles.quot(e);
    it.t = e - it.b * a.n_t;
  } else {  // causal rows: the longest first
    const int q = a.by_B.quot(li);
    it.b = li - q * a.B;
    it.t = a.n_t - 1 - q;
  }
  key_tiles(a.mask, it.b, a.n_t, it.t, it.r, it.f);
  return it;
}

// The tiles of this CTA one after another, across items.
struct Walk {
  int it = -1, j = 0;
  Item w;
  // 1: at the next tile, 0: no more, -1: the wait for an item ran out
  __device__ __forceinline__ int next(const Ring<Item>& ring, int* err, volatile int* abort_flag) {
    if (it >= 0 && ++j < w.r.y) return 1;
    if (!ring.get_thread(w, ++it, err, abort_flag)) return -1;
    j = w.r.x;
    return w.b >= 0;
  }
  __device__ __forceinline__ bool first() const { return j == w.r.x; }
  __device__ __forceinline__ bool last() const { return j == w.r.y - 1; }
};

template <int D, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1)
    masked_attn_dq_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_do,
                          const __grid_constant__ CUtensorMap tm_dqkv, const Args a) {
  pdl_trigger();
  using C = Cfg<D>;
  constexpr int QB = C::QB, NK = C::NK, NV = C::NV;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sQ = smem + C::Q_OFF;
  uint8_t* sK = smem + C::K_OFF;
  uint8_t* sV = smem + C::V_OFF;
  float* sST = reinterpret_cast<float*>(smem + C::ST_OFF);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* q_full = bars;            // [2]
  uint64_t* q_empty = bars + 2;       // [2]
  uint64_t* st_empty = bars + 6;      // [2]  row statistics read (16 warps)
  uint64_t* s_full = bars + 8;        // [2]  S computed
  uint64_t* k_full = bars + 10;       // [4]
  uint64_t* k_empty = bars + 14;      // [4]
  uint64_t* v_full = bars + 18;       // [4]
  uint64_t* v_empty = bars + 22;      // [4]
  uint64_t* dp_full = bars + 26;      // dP computed
  uint64_t* ds_full = bars + 27;      // dS written, dP read (16 warps)
  uint64_t* dq_full = bars + 28;      // dQ of an item complete
  uint64_t* dq_free = bars + 29;      // ... read (16 warps)
  uint64_t* out_full = bars + 30;     // dQ of an item staged (16 warps)
  uint64_t* ring_full = bars + 31;    // [kRing]
  uint64_t* ring_empty = bars + 35;   // [kRing]
  uint64_t* drain = bars + 39;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 40);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Ring<Item> ring{reinterpret_cast<Item*>(smem + C::ITEM_OFF), ring_full, ring_empty};

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&st_empty[i], kWarps);
      mbar_init(&s_full[i], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&ring_full[i], 1);
      mbar_init(&ring_empty[i], kConsumers);
    }
    mbar_init(dp_full, 1);
    mbar_init(ds_full, kWarps);
    mbar_init(dq_full, 1);
    mbar_init(dq_free, kWarps);
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
        int n = 0, q_issued = -1, k_issued = 0, v_issued = 0;
        bool ok = true;
        Walk x;
        for (int got; (got = x.next(ring, a.err, abort_flag)) != 0; ++n) {
          if (got < 0) { ok = false; break; }
          const int hk = a.by_group.quot(x.w.h);
          if (x.first()) {
            const int qb = x.it % QB;
            if (x.it >= QB && !bwait(&q_empty[qb], ((x.it / QB) - 1) & 1, a.err, abort_flag)) { ok = false; break; }
            if (x.it >= QB && !bwait(&st_empty[qb], ((x.it / QB) - 1) & 1, a.err, abort_flag)) { ok = false; break; }
            uint8_t* qd = sQ + qb * 2 * C::TILE;
            mbar_expect_tx(&q_full[qb], 2 * C::TILE + 1024);
            bulk_load(sST + qb * 256, a.ld + (((size_t)x.w.b * a.nh + x.w.h) * a.n_t + x.w.t) * (2 * BT), 1024, &q_full[qb]);
            load_tile<D>(qd, &tm_qkv, &q_full[qb], x.w.h * D, x.w.t * BT, x.w.b);
            load_tile<D>(qd + C::TILE, &tm_do, &q_full[qb], x.w.h * D, x.w.t * BT, x.w.b);
            q_issued = x.it;
          }
          const int ks = n % NK, vs = n % NV;
          if (n >= NK && !bwait(&k_empty[ks], ((n / NK) - 1) & 1, a.err, abort_flag)) { ok = false; break; }
          mbar_expect_tx(&k_full[ks], C::TILE);
          load_tile<D>(sK + ks * C::TILE, &tm_qkv, &k_full[ks], (a.nh + hk) * D, x.j * BT, x.w.b);
          k_issued = n + 1;
          if (n >= NV && !bwait(&v_empty[vs], ((n / NV) - 1) & 1, a.err, abort_flag)) { ok = false; break; }
          mbar_expect_tx(&v_full[vs], C::TILE);
          load_tile<D>(sV + vs * C::TILE, &tm_qkv, &v_full[vs], (a.nh + a.nkv + hk) * D, x.j * BT, x.w.b);
          v_issued = n + 1;
        }
        if (!ok) {
          for (int u = max(0, q_issued - QB + 1); u <= q_issued; ++u) drain_wait(&q_full[u % QB], (u / QB) & 1);
          for (int u = max(0, k_issued - NK); u < k_issued; ++u) drain_wait(&k_full[u % NK], (u / NK) & 1);
          for (int u = max(0, v_issued - NV); u < v_issued; ++u) drain_wait(&v_full[u % NV], (u / NV) & 1);
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      if (elect_one()) {
        // ---------------------------------------------------------------- MMA
        bool ok = true;
        int n = 0;
        Walk cur, nxt;
        auto issue_s = [&](const Walk& x, int u) -> bool {
          const int qb = x.it % QB;
          if (x.first() && !bwait(&q_full[qb], (x.it / QB) & 1, a.err, abort_flag)) return false;
          if (!bwait(&k_full[u % NK], (u / NK) & 1, a.err, abort_flag)) return false;
          tc_fence_after();
          mma_abt<D>(tmem + C::T_S + (u & 1) * 128, smem_u32(sQ + qb * 2 * C::TILE), smem_u32(sK + (u % NK) * C::TILE));
          umma_commit(&s_full[u & 1]);
          return true;
        };
        auto issue_dp = [&](const Walk& x, int u) -> bool {
          const int qb = x.it % QB;
          if (!bwait(&v_full[u % NV], (u / NV) & 1, a.err, abort_flag)) return false;
          tc_fence_after();
          mma_abt<D>(tmem + C::T_DP, smem_u32(sQ + qb * 2 * C::TILE + C::TILE), smem_u32(sV + (u % NV) * C::TILE));
          umma_commit(dp_full);
          umma_commit(&v_empty[u % NV]);
          if (x.last()) umma_commit(&q_empty[qb]);  // every product of this item that reads Q or dO is issued
          return true;
        };
        int more = nxt.next(ring, a.err, abort_flag);
        ok = more >= 0 && (more == 0 || (issue_s(nxt, 0) && issue_dp(nxt, 0)));
        while (ok && more) {
          cur = nxt;
          more = nxt.next(ring, a.err, abort_flag);
          if (more < 0) { ok = false; break; }
          // one Q buffer: the next item's Q can only be loaded once this item's products are done with it,
          // and this tile's dQ should not wait for that load
          const bool early = more && (QB == 2 || nxt.it == cur.it);
          if (early && !issue_s(nxt, n + 1)) { ok = false; break; }
          if (!bwait(ds_full, n & 1, a.err, abort_flag)) { ok = false; break; }
          if (early && !issue_dp(nxt, n + 1)) { ok = false; break; }
          if (cur.first() && cur.it > 0 && !bwait(dq_free, (cur.it - 1) & 1, a.err, abort_flag)) { ok = false; break; }
          tc_fence_after();
          mma_tmem_b<D, 32>(tmem + C::T_DQ, tmem + C::T_S + (n & 1) * 128, smem_u32(sK + (n % NK) * C::TILE),
                        !cur.first());
          // the K stage of an item's last tile becomes the staging tile of its dQ, which then releases it
          if (cur.last()) umma_commit(dq_full);
          else umma_commit(&k_empty[n % NK]);
          if (more && !early && !(issue_s(nxt, n + 1) && issue_dp(nxt, n + 1))) { ok = false; break; }
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
      const int n_items = a.B * a.nh * a.n_t;
      Item w;
      for (int r = 0, k = 0;; ++r) {
        const int item = snake_item(r);
        if (item < n_items) {
          w = decode(a, item);
          if (w.r.x >= w.r.y) {
            const size_t width = (size_t)(a.nh + 2 * a.nkv) * D;
            zero_rows<2 * D>(a.dqkv + ((size_t)w.b * a.S + w.t * BT) * width + (size_t)w.h * D, 2 * width,
                             min(BT, a.S - w.t * BT));
            continue;
          }
        } else {
          w.b = -1;
        }
        if (!ring.put_warp(w, k++, a.err, abort_flag) || w.b < 0) break;
      }
    } else {
      // ---------------------------------------------------------------- stores of staged dQ tiles
      int n = 0, it = 0;
      Item w;
      for (int u = 0; ring.get_warp(w, u, a.err, abort_flag) && w.b >= 0; ++u) {
        n += w.r.y - w.r.x;
        if (!wwait(out_full, it & 1, a.err, abort_flag)) break;
        if (lane == 0) {
          const int ks = (n - 1) % NK;
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_store_3d(&tm_dqkv, sK + ks * C::TILE + c * 16384, w.h * D + c * 64, w.t * BT, w.b);
          bulk_commit();
          bulk_wait_read<0>();
          mbar_arrive(&k_empty[ks]);
        }
        __syncwarp();
        ++it;
      }
      if (lane == 0) bulk_wait<0>();
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------------ dS, dQ store
    reg_inc<104>();
    const int part = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const Score k = a.score;
    int n = 0, it = 0;
    bool ok = true;
    // dQ of item number `of`, whose last tile was number `last`: TMEM -> the K stage of that tile, for the store warp
    auto drain_dq = [&](int of, int last) -> bool {
      if (!wwait(dq_full, of & 1, a.err, abort_flag)) return false;
      tc_fence_after();
      uint32_t v[D / 4];
      tmem_ld(tmem + C::T_DQ + lane_off + part * (D / 4), v);
      tmem_wait_ld();
      warp_arrive(dq_free);
      stage_row(sK + (last % NK) * C::TILE, 16384, row, part * (D / 4), v, a.scale);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(out_full);
      return true;
    };
    int last = -1;  // last tile of the item whose dQ is still in TMEM
    Item w;
    for (int u = 0; ok && (ok = ring.get_warp(w, u, a.err, abort_flag)) && w.b >= 0; ++u) {
      const int i = w.t * BT + row;
      int start = 0, end = i + 1;
      if (a.mask.rows) {
        const int* tr = a.mask.rows + ((size_t)w.b * a.n_t + w.t) * (4 * BT) + row;
        start = tr[0];
        end = tr[BT];
      }
      float slope = 0.f;
      if (BIAS) slope = a.slopes[w.h] * kLog2e;
      const int qb = it % QB;
      if (!wwait(&q_full[qb], (it / QB) & 1, a.err, abort_flag)) { ok = false; break; }
      const float2 st = make_float2(sST[qb * 256 + row], sST[qb * 256 + BT + row]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&st_empty[qb]);
      for (int j = w.r.x; j < w.r.y; ++j, ++n) {
        const uint32_t t_s = tmem + C::T_S + (n & 1) * 128 + lane_off + part * 32;
        if (!wwait(&s_full[n & 1], (n >> 1) & 1, a.err, abort_flag)) { ok = false; break; }
        tc_fence_after();
        float pf[32];  // P (1 - tanh^2)
        {
          uint32_t s[32];
          tmem_ld(t_s, s);
          tmem_wait_ld();
          if (CAP) cap_in_place(s, k);
          const int j0 = j * BT + part * 32;  // key of column 0
          const float dist = (float)(j0 - i);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float2 x = pair(s[e], s[e + 1]), f;
            if (CAP) {
              f = fma2(mul2(x, pair(-1.f)), x, pair(1.f));  // 1 - tanh^2
              x = mul2(x, pair(k.cap));
            }
            if (BIAS) {
              if (!CAP) x = mul2(x, pair(k.mul));
              x.x = fmaf(-slope, fabsf(dist + (float)e), x.x);
              x.y = fmaf(-slope, fabsf(dist + (float)(e + 1)), x.y);
            }
            x = (CAP || BIAS) ? add2(x, pair(st.x)) : fma2(x, pair(k.mul), pair(st.x));
            x = exp2_pair(x);
            if (CAP) x = mul2(x, f);
            pf[e] = x.x;
            pf[e + 1] = x.y;
          }
          if (j < w.f.x || j >= w.f.y) {
            const uint32_t seen = seen_bits(start, end, j0);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen & (1u << e))) pf[e] = 0.f;
          }
        }
        // the previous item's dQ leaves here: its last product ran while this tile's P was computed
        if (last >= 0) {
          if (!drain_dq(it - 1, last)) { ok = false; break; }
          last = -1;
        }
        if (!wwait(dp_full, n & 1, a.err, abort_flag)) { ok = false; break; }
        tc_fence_after();
        {
          uint32_t dp[32];
          tmem_ld(tmem + C::T_DP + lane_off + part * 32, dp);
          tmem_wait_ld();
          uint32_t ds[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 v = mul2(make_float2(pf[2 * e], pf[2 * e + 1]), add2(pair(dp[2 * e], dp[2 * e + 1]), pair(st.y)));
            ds[e] = pack_bf16x2(v.x, v.y);
          }
          tmem_st_32x32b_x16(t_s, ds);
        }
        tmem_wait_st();
        warp_arrive(ds_full);
      }
      if (!ok) break;
      last = n - 1;
      ++it;
    }
    if (ok && last >= 0) drain_dq(it - 1, last);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

constexpr int kStatRows = 8;

// ld[b, h, tile, 0 / 1, row] = -LSE log2 e / -Delta; -inf and 0 for a row that takes no part.  A CTA has 8 tokens
// of one batch entry, all heads: neighbouring threads read neighbouring 16 bytes, the d / 8 threads of a (token, head)
// add up with shuffles, and the results leave through shared memory as 32-byte runs per head.
template <int D>
__global__ void __launch_bounds__(256)
    row_stats_kernel(const __nv_bfloat16* __restrict__ dout, long do_ss, long do_sb, const __nv_bfloat16* __restrict__ out,
                     const float* __restrict__ lse, int S, int nh, int n_t, float* __restrict__ ld) {
  pdl_trigger();
  constexpr int G = D / 8;
  extern __shared__ float s_delta[];  // [nh][kStatRows + 1]
  const int blocks = n_t * (BT / kStatRows);
  const int b = blockIdx.x / blocks, row0 = (blockIdx.x % blocks) * kStatRows;
  const int per_row = nh * G, units = kStatRows * per_row;
  pdl_wait();
  // every thread of a warp takes part in the shuffles: units and the block size are multiples of the warp size
#pragma unroll 4
  for (int u = threadIdx.x; u < units; u += 256) {
    const int r = u / per_row, c = u - r * per_row;
    const int i = row0 + r;
    float acc = 0.f;
    if (i < S) {
      const uint4 x = *reinterpret_cast<const uint4*>(dout + b * do_sb + i * do_ss + c * 8);
      const uint4 y = *reinterpret_cast<const uint4*>(out + ((size_t)b * S + i) * ((size_t)nh * D) + c * 8);
      const uint32_t* xw = reinterpret_cast<const uint32_t*>(&x);
      const uint32_t* yw = reinterpret_cast<const uint32_t*>(&y);
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const float2 f = unpack_bf16x2(xw[z]), g = unpack_bf16x2(yw[z]);
        acc = fmaf(f.x, g.x, fmaf(f.y, g.y, acc));
      }
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (c % G == 0) s_delta[(c / G) * (kStatRows + 1) + r] = acc;
  }
  __syncthreads();
  for (int u = threadIdx.x; u < nh * kStatRows; u += 256) {
    const int h = u / kStatRows, r = u % kStatRows, i = row0 + r;
    const float l = i < S ? lse[((size_t)b * nh + h) * S + i] : -INFINITY;
    const bool none = l == -INFINITY;
    float* p = ld + (((size_t)b * nh + h) * n_t + row0 / BT) * (2 * BT) + row0 % BT + r;
    p[0] = none ? -INFINITY : -l * kLog2e;
    p[BT] = none ? 0.f : -s_delta[h * (kStatRows + 1) + r];
  }
}

template <int D>
int row_stats(const AttnCall& c, const void* dout, long do_ss, long do_sb, const void* out, const float* lse, float* ld,
              cudaStream_t stream) {
  const int n_t = (c.S + BT - 1) / BT;
  const long grid = (long)c.B * n_t * (BT / kStatRows);
  const size_t smem = (size_t)c.nh * (kStatRows + 1) * sizeof(float);
  if (grid > INT_MAX || smem > 200 * 1024) return -4;
  auto k = row_stats_kernel<D>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
  }
  launch_early(0, k, (unsigned)grid, 256, smem, stream, static_cast<const __nv_bfloat16*>(dout), do_ss, do_sb,
           static_cast<const __nv_bfloat16*>(out), lse, c.S, c.nh, n_t, ld);
  return (int)cudaGetLastError();
}

template <int D, bool CAP, bool BIAS>
int launch(const CUtensorMap& tq, const CUtensorMap& to, const CUtensorMap& td, const Args& a, int grid, cudaStream_t stream) {
  auto k = masked_attn_dq_kernel<D, CAP, BIAS>;
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM);
  if (e != cudaSuccess) return (int)e;
  launch_early(0, k, grid, kThreads, Cfg<D>::SMEM, stream, tq, to, td, a);
  return (int)cudaGetLastError();
}

}  // namespace dq
}  // namespace mattn

int masked_attn_dq(const AttnCall& c, const void* dout, long do_ss, long do_sb, const void* out, const float* lse,
                   float* ld, void* dqkv, int* err, int num_sms, cudaStream_t stream) {
  using namespace mattn;
  const int n_t = (c.S + BT - 1) / BT;
  const long items = (long)c.B * c.nh * n_t;
  if (items > INT_MAX / 2) return -1;
  if (c.d != 64 && c.d != 128) return -2;
  int rc = c.d == 64 ? dq::row_stats<64>(c, dout, do_ss, do_sb, out, lse, ld, stream)
                     : dq::row_stats<128>(c, dout, do_ss, do_sb, out, lse, ld, stream);
  if (rc) return rc;
  CUtensorMap tq, to, td;
  rc = make_tmap_bf16_3d(&tq, c.qkv, c.B, c.S, (long)(c.nh + 2 * c.nkv) * c.d, c.qkv_ss, c.qkv_sb, 64, BT);
  if (rc) return rc - 10;
  rc = make_tmap_bf16_3d(&to, dout, c.B, c.S, (long)c.nh * c.d, do_ss, do_sb, 64, BT);
  if (rc) return rc - 20;
  const long width = (long)(c.nh + 2 * c.nkv) * c.d;
  rc = make_tmap_bf16_3d(&td, dqkv, c.B, c.S, width, width, width * c.S, 64, BT);
  if (rc) return rc - 30;
  dq::Args a;
  a.B = c.B;
  a.S = c.S;
  a.nh = c.nh;
  a.nkv = c.nkv;
  a.n_t = n_t;
  a.by_nh = FastDiv(c.nh);
  a.by_B = FastDiv(c.B);
  a.by_tiles = FastDiv(n_t);
  a.by_group = FastDiv(c.nh / c.nkv);
  a.mask = Mask{c.rows, static_cast<const int4*>(c.qstat), static_cast<const int4*>(c.kstat), c.order_q};
  a.slopes = c.slopes;
  a.score = score_constants(c.scale, c.cap);
  a.scale = c.scale;
  a.ld = ld;
  a.dqkv = static_cast<__nv_bfloat16*>(dqkv);
  a.err = err;
  const int grid = (int)std::max(1L, std::min(items, (long)num_sms));
  const bool cap = c.cap > 0.f, bias = c.slopes != nullptr;
  if (c.d == 64) {
    if (cap) return bias ? dq::launch<64, true, true>(tq, to, td, a, grid, stream) : dq::launch<64, true, false>(tq, to, td, a, grid, stream);
    return bias ? dq::launch<64, false, true>(tq, to, td, a, grid, stream) : dq::launch<64, false, false>(tq, to, td, a, grid, stream);
  }
  if (c.d == 128) {
    if (cap) return bias ? dq::launch<128, true, true>(tq, to, td, a, grid, stream) : dq::launch<128, true, false>(tq, to, td, a, grid, stream);
    return bias ? dq::launch<128, false, true>(tq, to, td, a, grid, stream) : dq::launch<128, false, false>(tq, to, td, a, grid, stream);
  }
  return -2;
}

}  // namespace mmb
