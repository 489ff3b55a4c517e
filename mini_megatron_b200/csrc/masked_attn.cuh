// Shared parts of the masked attention kernels (masked_attn_fwd.cu,
// masked_attn_dq.cu, masked_attn_dkv.cu): the mask, the score transform, bounded
// waits and the order of work items.
//
// Scores in log2 units, query i, key j, head h, C = cap * log2 e:
//
//   x_ij = C tanh(s q_i.k_j / cap)  or  s log2 e (q_i.k_j),   minus  slope_h log2 e |i - j|
//   visible iff start_i <= j < end_i                          (document_plan.cu; causal: 0 and i + 1)
//
// tanh u of a warp whose scores all have |u| <= 1 (the cap well above them, the usual case) is u times a polynomial
// in u^2: it runs on the FMA pipe, while 1 - 2 / (1 + e^{2u}), used otherwise, takes two of the three MUFU
// operations of a score, and those bound the capped kernels (16 a cycle and SM; forward of 4 x 2048 tokens, 16 heads
// of 128, cap 30: 129 us with the polynomial, 152 without; dQ 122 and 141, dK and dV 173 and 195).  Both are
// exact to a few 2^-23.  The single-instruction tanh approximation is off by up to 2^-11 relative, which a cap of 50
// turns into 0.02 in the exponent; it is not used.
//
// Roundings to 16 bits, besides the outputs: P, as operand of P V and of dV, and dS, as operand of dQ and dK.  The other
// operand of each of these products is bf16 and the tensor cores take pairs of one type; in 32 bits (tf32) the
// products would take twice the time and P and dS twice the TMEM columns, which are all in use.  Delta is taken from ctx as
// it was returned, rounded.  The forward's epilogue has the unrounded O and could write what the rounding took off as a
// second bf16 tensor for row_stats to add (25 MB each way at 16 x 1024 tokens, 12 heads of 64: about 8 us of 210); it does
// not, because the backward is a function of ctx and lse alone.  Against 64 bits the outputs are
// off by 0.0021 to 0.0036 (norm of the error over the norm): one rounding of the outputs makes 0.0017, P and dS 0.0016, Delta
// 0.0005 with even weights to 0.0019 with sharp ones.
//
// These kernels, row_stats, rotary and the plans are launched early (launch_early): barriers, TMEM and the first
// instructions are set up behind the predecessor's last CTAs.  Short calls are made of that: forward and backward of 2
// rows of 77 tokens 28.7 -> 22.5 us, S = 16384 719 -> 702 us.  The predecessor may be any kernel that triggers, plainly
// launched ones among them; all of its CTAs have started by then.  An early CTA holds all of its SM's TMEM while it
// waits; the predecessor cannot be kept from its own by that, because no kernel that uses TMEM fits beside 200 KB
// of shared memory on one SM.
#pragma once
#include "common.cuh"
#include "ops.h"

#include <algorithm>
#include <climits>

namespace mmb {
namespace mattn {

constexpr int BT = 128;  // rows of every query and key tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

struct Mask {
  const int* rows;    // [B, n_t, 4, 128] start, end; the queries that see the token as a key (tile-padded); nullptr: causal
  const int4* qstat;  // [B, n_t] {min start, max end, max start, min end}
  const int4* kstat;  // [B, n_t] the same of the query intervals
  const int* order;   // this kernel's tiles of all rows, heaviest first, or nullptr: by position
};

// Tiles [x, y) of the other side that a tile with these bounds needs, and those of them that need no mask: every row
// sees all of the tile.  (Rows behind the end of the sequence do not count: what they read is zero.)
// Both are kept within the row, and entries of the order within the batch, so that a table that was captured but not
// yet written sends nothing out of range.
__device__ __forceinline__ int2 needed_tiles(const int4& q, int n_t) {
  return q.y <= 0 ? make_int2(0, 0) : make_int2(max(q.x / BT, 0), min((q.y - 1) / BT + 1, n_t));
}
__device__ __forceinline__ int ordered(const int* order, int k, int n) { return min(max(order[k], 0), n - 1); }
__device__ __forceinline__ int2 whole_tiles(const int4& q) { return make_int2((q.z + BT - 1) / BT, q.w / BT); }

// Key tiles of query tile t of row b.
__device__ __forceinline__ void key_tiles(const Mask& m, int b, int n_t, int t, int2& need, int2& whole) {
  if (!m.rows) {
    need = make_int2(0, t + 1);
    whole = make_int2(0, t);
    return;
  }
  const int4 q = m.qstat[(size_t)b * n_t + t];
  need = needed_tiles(q, n_t);
  whole = whole_tiles(q);
}
// Query tiles of key tile t of row b.
__device__ __forceinline__ void query_tiles(const Mask& m, int b, int n_t, int t, int2& need, int2& whole) {
  if (!m.rows) {
    need = make_int2(t, n_t);
    whole = make_int2(t + 1, n_t);
    return;
  }
  const int4 q = m.kstat[(size_t)b * n_t + t];
  need = needed_tiles(q, n_t);
  whole = whole_tiles(q);
}
// Which of 32 consecutive rows or columns from `first` on lie in [lo, hi).
__device__ __forceinline__ uint32_t seen_bits(int lo, int hi, int first) {
  const int l = min(max(lo - first, 0), 32), h = min(max(hi - first, 0), 32);
  return (h >= 32 ? 0xffffffffu : (1u << h) - 1u) & ~(l >= 32 ? 0xffffffffu : (1u << l) - 1u);
}

// Item of this CTA in round `r`: every other round runs backwards over the CTAs, so that with items
// sorted by weight the CTA with the heaviest item of one round takes the lightest of the next.
__device__ __forceinline__ int snake_item(int r) {
  return r * (int)gridDim.x + ((r & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
}

// n / d for 0 <= n < 2^31 by a multiplication (the round-up method: m = ceil(2^(31 + l) / d), 2^(l-1) < d <= 2^l).
struct FastDiv {
  uint32_t m, l, d;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : l(0), d(div) {
    while ((1ull << l) < div) ++l;
    m = (uint32_t)(((1ull << (31 + l)) + div - 1) / div);
  }
  __device__ __forceinline__ int quot(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> (31 + l)); }
};

// Work items travel from one scheduling thread (forward) or warp (backward) to the roles through a ring in shared memory: decoding an item
// (divisions, loads of the mask's tile tables) takes about a thousand cycles, which every role would otherwise
// spend between two items.
constexpr int kRing = 4;
template <typename Item>
struct Ring {
  Item* items;
  uint64_t* full;   // [kRing] 1 arrival
  uint64_t* empty;  // [kRing] one arrival per consumer
  // consumer side, item number k: a whole warp / one thread
  __device__ __forceinline__ bool get_warp(Item& w, int k, int* err, volatile int* abort_flag) const;
  __device__ __forceinline__ bool get_thread(Item& w, int k, int* err, volatile int* abort_flag) const;
  // producer side: one thread / a whole warp
  __device__ __forceinline__ bool put(const Item& w, int k, int* err, volatile int* abort_flag) const;
  __device__ __forceinline__ bool put_warp(const Item& w, int k, int* err, volatile int* abort_flag) const;
};

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}

__device__ __forceinline__ float2 exp2_pair(float2 x) { return make_float2(fast_exp2(x.x), fast_exp2(x.y)); }
__device__ __forceinline__ float2 pair(float a) { return make_float2(a, a); }
__device__ __forceinline__ float2 pair(uint32_t a, uint32_t b) {
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}

// Constants of the score transform.
struct Score {
  float mul;    // plain: s log2 e;  capped: s / cap (u = mul q.k)
  float twice;  // capped: 2 s log2 e / cap (e^{2u} = 2^(twice q.k))
  float cap;    // C
};

// tanh u for |u| <= 1: u times a polynomial of degree 6 in u^2, fitted for the least relative error (1.6e-7).
__device__ __forceinline__ float2 tanh_small(float2 u) {
  const float2 z = mul2(u, u);
  float2 p = fma2(z, pair(1.041017706e-03f), pair(-6.203362253e-03f));
  p = fma2(p, z, pair(2.028995939e-02f));
  p = fma2(p, z, pair(-5.345701799e-02f));
  p = fma2(p, z, pair(1.332520396e-01f));
  p = fma2(p, z, pair(-3.333283961e-01f));
  p = fma2(p, z, pair(9.999999404e-01f));
  return mul2(u, p);
}
// tanh of a pair of scores.
template <bool SMALL>
__device__ __forceinline__ float2 cap_tanh(float2 s, const Score& k) {
  if constexpr (SMALL) return tanh_small(mul2(s, pair(k.mul)));
  const float2 e = add2(exp2_pair(mul2(s, pair(k.twice))), pair(1.f));
  return fma2(make_float2(rcp_approx(e.x), rcp_approx(e.y)), pair(-2.f), pair(1.f));
}
// Whether every |u| of the warp's N scores a thread is at most 1.  The maximum passes over a NaN, which may so be taken for
// a small score; either form of tanh keeps it a NaN.
template <int N>
__device__ __forceinline__ bool cap_small(const uint32_t (&s)[N], const Score& k) {
  float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < N; c += 2)
    m[(c / 2) & 3] = max3(m[(c / 2) & 3], fabsf(__uint_as_float(s[c])), fabsf(__uint_as_float(s[c + 1])));
  return __all_sync(0xffffffffu, max3(fmaxf(m[0], m[1]), m[2], m[3]) * k.mul <= 1.f) != 0;
}

// The warp's scores replaced by their tanh u.
template <int N>
__device__ __forceinline__ void cap_in_place(uint32_t (&s)[N], const Score& k) {
  if (cap_small(s, k)) {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const float2 t = cap_tanh<true>(pair(s[c], s[c + 1]), k);
      s[c] = __float_as_uint(t.x);
      s[c + 1] = __float_as_uint(t.y);
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const float2 t = cap_tanh<false>(pair(s[c], s[c + 1]), k);
      s[c] = __float_as_uint(t.x);
      s[c + 1] = __float_as_uint(t.y);
    }
  }
}

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// One thread of the (converged) warp.  tcgen05.mma and TMA take their descriptors from uniform registers:
// behind elect.sync the compiler knows that a single thread is left and moves them there directly, behind a
// test of the lane index it has to assume several threads with different values and issues each instruction
// from a loop (measured in the forward kernel: 8 products took 1100 cycles to issue).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(p));
  return p != 0;
}

// Bounded wait on an mbarrier phase.  The clock is read only after many polls: a read of the
// global timer costs more than most of these waits.
__device__ __forceinline__ bool bwait(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag) {
  unsigned long long t0 = 0;
  for (uint32_t n = 1;; ++n) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((n & 255u) == 0) {
      if (*abort_flag) return false;
      const unsigned long long now = globaltimer();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > kWaitTimeoutNs) {
        if (err) atomicExch(err, (int)kErrAttnWait);
        *abort_flag = 1;
        return false;
      }
    }
  }
}

// Warp-wide: the warp goes on only if every lane saw the phase complete.
__device__ __forceinline__ bool wwait(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag) {
  const bool ok = bwait(bar, parity, err, abort_flag);
  return __all_sync(0xffffffffu, ok) != 0;
}

// Bounded wait used while winding down after an abort (does not look at the abort flag).
__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer();
  while (!mbar_try_wait(bar, parity) && globaltimer() - t0 < 20000000ull) {
  }
}

template <typename Item>
__device__ __forceinline__ bool Ring<Item>::get_thread(Item& w, int k, int* err, volatile int* abort_flag) const {
  if (!bwait(&full[k % kRing], (k / kRing) & 1, err, abort_flag)) return false;
  w = items[k % kRing];
  mbar_arrive(&empty[k % kRing]);
  return true;
}
template <typename Item>
__device__ __forceinline__ bool Ring<Item>::get_warp(Item& w, int k, int* err, volatile int* abort_flag) const {
  if (!wwait(&full[k % kRing], (k / kRing) & 1, err, abort_flag)) return false;
  w = items[k % kRing];
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&empty[k % kRing]);
  return true;
}
template <typename Item>
__device__ __forceinline__ bool Ring<Item>::put(const Item& w, int k, int* err, volatile int* abort_flag) const {
  if (k >= kRing && !bwait(&empty[k % kRing], ((k / kRing) - 1) & 1, err, abort_flag)) return false;
  items[k % kRing] = w;
  mbar_arrive(&full[k % kRing]);
  return true;
}

template <typename Item>
__device__ __forceinline__ bool Ring<Item>::put_warp(const Item& w, int k, int* err, volatile int* abort_flag) const {
  if (k >= kRing && !wwait(&empty[k % kRing], ((k / kRing) - 1) & 1, err, abort_flag)) return false;
  if ((threadIdx.x & 31) == 0) {
    items[k % kRing] = w;
    mbar_arrive(&full[k % kRing]);
  }
  __syncwarp();
  return true;
}

// One arrival per warp on `bar`, after every lane's tcgen05 loads / stores are ordered before it.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// A [rows, 128-byte chunks] tile of D columns, as CHUNKS boxes of 64 columns x 128 rows.
template <int D>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int col, int row,
                                          int batch) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c) tma_load_3d(dst + c * 16384, map, bar, col + 64 * c, row, batch);
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
               : "memory");
}

// N fp32 values of one row, from column col0 on, as bf16 into a staged tile (chunks of 64 columns, `chunk`
// bytes apart, rows of 128 bytes in the 128-byte swizzle) for a tensor store.  A thread owns a row of an
// accumulator, so direct stores would touch 32 rows per instruction and hold the load/store pipe, and
// every barrier poll behind it, for thousands of cycles per tile.
template <int N>
__device__ __forceinline__ void stage_row(uint8_t* tile, int chunk, int row, int col0, const uint32_t (&v)[N],
                                          float mul) {
#pragma unroll
  for (int u = 0; u < N / 8; ++u) {
    const int unit = col0 / 8 + u;
    uint4 w;
    w.x = pack_bf16x2(__uint_as_float(v[8 * u + 0]) * mul, __uint_as_float(v[8 * u + 1]) * mul);
    w.y = pack_bf16x2(__uint_as_float(v[8 * u + 2]) * mul, __uint_as_float(v[8 * u + 3]) * mul);
    w.z = pack_bf16x2(__uint_as_float(v[8 * u + 4]) * mul, __uint_as_float(v[8 * u + 5]) * mul);
    w.w = pack_bf16x2(__uint_as_float(v[8 * u + 6]) * mul, __uint_as_float(v[8 * u + 7]) * mul);
    *reinterpret_cast<uint4*>(tile + (unit >> 3) * chunk + row * 128 + (((unit & 7) ^ (row & 7)) << 4)) = w;
  }
}

// 128 x 128 (+)= A [128 x D] B [128 x D]^T, both K-major in shared memory.
template <int D>
__device__ __forceinline__ void mma_abt(uint32_t dst, uint32_t a_addr, uint32_t b_addr) {
  constexpr uint32_t idesc = make_idesc_bf16(BT, BT, false, false);
  const uint64_t ad = make_sdesc_sw128(a_addr, 16, 1024), bd = make_sdesc_sw128(b_addr, 16, 1024);
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
    umma_bf16_ss(dst, ad + off, bd + off, idesc, k != 0 ? 1u : 0u);
  }
}

// 128 x D (+)= A [128 x 128, bf16 in TMEM] B [128 x D] (rows are the reduction: MN-major).  A's 128
// columns lie in runs of RUN (RUN / 2 TMEM columns) that start STRIDE TMEM columns apart.  K0, K1: part of the
// reduction, in steps of 16.
template <int D, int RUN, int STRIDE = 32, int K0 = 0, int K1 = BT / 16>
__device__ __forceinline__ void mma_tmem_b(uint32_t dst, uint32_t a_tmem, uint32_t b_addr, bool acc) {
  constexpr int PER = RUN / 16;
  constexpr uint32_t idesc = make_idesc_bf16(BT, D, false, true);
  const uint64_t bd = make_sdesc_sw128(b_addr, 16384, 1024);
#pragma unroll
  for (int k = K0; k < K1; ++k)
    umma_bf16_ts(dst, a_tmem + (k / PER) * STRIDE + (k % PER) * 8, bd + (uint64_t)(k * (2048 >> 4)), idesc,
                 (acc || k != 0) ? 1u : 0u);
}

__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld_32x32b_x32(taddr, r); }
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld_32x32b_x16(taddr, r); }

// `rows` rows of BYTES bytes, `stride` bytes apart, set to zero by one warp.
template <int BYTES>
__device__ __forceinline__ void zero_rows(void* p, size_t stride, int rows) {
  constexpr int PER = BYTES / 16;
  const int lane = threadIdx.x & 31;
  for (int u = lane; u < rows * PER; u += 32)
    *reinterpret_cast<uint4*>(static_cast<char*>(p) + (u / PER) * stride + (u % PER) * 16) = make_uint4(0u, 0u, 0u, 0u);
}

// N values of one row set to zero.
template <int N>
__device__ __forceinline__ void store_zero(__nv_bfloat16* p) {
#pragma unroll
  for (int u = 0; u < N / 8; ++u) reinterpret_cast<uint4*>(p)[u] = make_uint4(0u, 0u, 0u, 0u);
}

}  // namespace mattn

// Host-side description of one call (ops.h declares the launchers).
inline mattn::Score score_constants(float scale, float cap) {
  if (cap > 0.f) return {scale / cap, 2.f * scale * mattn::kLog2e / cap, cap * mattn::kLog2e};
  return {scale * mattn::kLog2e, 0.f, 0.f};
}

}  // namespace mmb
