// Positions and visible key intervals of packed rows.
//
// A row of S tokens holds documents one after another and possibly padding at
// its end.  Token i sees the keys [start_i, end_i) of its own row:
//
//   start_i = the largest document start <= i
//   end_i   = i + 1, or, while every token from start_i to i is marked as
//             prefix, the first index after i that is unmarked, begins a
//             document, is padding, or is S
//   position_i = i - start_i
//
// Padding sees nothing: start = end = position = 0.  Seen from the keys, key j is
// visible to the queries [j, document end), or, as part of a prefix, to its whole
// document: an interval again.  All of it comes from scans of one row: a running
// maximum of document starts, a running maximum of unmarked indices (a token is in
// its prefix iff that is < start_i), and running minima from the right of the
// document starts and of the indices that stop a prefix.
//
// For the attention kernels the same pass writes tile-padded copies of both intervals
// and, for every 128-token tile, the extremes of their bounds: which key tiles a query
// tile needs, which query tiles a key tile, and which of them need no mask.
//
// One cluster of 1 to 8 CTAs per row, the row cut into as many chunks; a
// thread owns 4 consecutive tokens, so a warp owns one 128-token tile and the
// tile statistics are warp reductions.  Each CTA first reduces its chunk, the
// chunk results cross the cluster through distributed shared memory, and a
// second sweep (right to left) scans and writes.  The work is a few bytes per
// token: latency bounds it, so the row is spread over CTAs as soon as one CTA
// would need more than one sweep step (4096 tokens).  8 x 32768 tokens: 10.0 us and 4.8 us for the
// order (2 x 257: 4.8 us), against 0.9 us for the bytes alone.
#include "common.cuh"
#include "ops.h"

#include <algorithm>
#include <climits>

namespace mmb {
namespace docplan {

constexpr int kThreads = 1024;
constexpr int kPer = 4;                      // tokens per thread: 32 lanes x 4 = one 128-token tile per warp
constexpr int kStep = kThreads * kPer;       // 4096 tokens per sweep step
constexpr int kMaxCtas = 8;                  // portable cluster size
constexpr int kMaxSteps = 64;                // per CTA: rows of up to 2 Mi tokens

struct Args {
  const long* ids;        // [B, S] tokens or document ids
  long ld_ids;
  long eod;
  int by_change;          // 1: a document starts where the id changes; 0: after a token equal to eod
  const uint8_t* marks;   // [B, S] prefix marks or nullptr
  long ld_marks;
  const int* lengths;     // [B] or nullptr
  int S, n_t, chunk;      // chunk: tokens per CTA (a multiple of kStep)
  int* positions;         // [B, S]
  int* start;
  int* end;
  int* rows;              // [B, n_t, 4, 128] start, end; first and one past the last query that sees the token
  int4* qstat;            // [B, n_t] {min start, max end, max start, min end}; no visible key: {INT_MAX, 0, ..}
  int4* kstat;            // [B, n_t] the same of the query intervals
};

struct alignas(16) Agg {
  int ds, lu, stop, nf;  // max document start, max unmarked index, min stopping index, min document start
};

__device__ __forceinline__ int warp_max_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = max(v, u);
  }
  return v;
}
__device__ __forceinline__ int warp_min_scan_right(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_down_sync(0xffffffffu, v, o);
    if (lane + o < 32) v = min(v, u);
  }
  return v;
}

// First (document start) and plain (unmarked or padding) flags of the thread's four tokens.
__device__ __forceinline__ void load_flags(const Args& a, int b, int i0, int len, bool (&first)[kPer],
                                           bool (&plain)[kPer]) {
  long id[kPer] = {0, 0, 0, 0};
  uint8_t mark[kPer] = {0, 0, 0, 0};
  long prev = 0;
  const bool whole = i0 + kPer <= a.S;
  if (i0 < a.S) {
    const long* p = a.ids + b * a.ld_ids + i0;
    if (i0 > 0) prev = p[-1];
    if (whole && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      const longlong2 u = *reinterpret_cast<const longlong2*>(p), v = *reinterpret_cast<const longlong2*>(p + 2);
      id[0] = u.x;
      id[1] = u.y;
      id[2] = v.x;
      id[3] = v.y;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (i0 + e < a.S) id[e] = p[e];
    }
  }
  if (a.marks && i0 < len) {
    const uint8_t* p = a.marks + b * a.ld_marks + i0;
    if (whole && (reinterpret_cast<uintptr_t>(p) & 3) == 0) {
      const uchar4 u = *reinterpret_cast<const uchar4*>(p);
      mark[0] = u.x;
      mark[1] = u.y;
      mark[2] = u.z;
      mark[3] = u.w;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (i0 + e < a.S) mark[e] = p[e];
    }
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int i = i0 + e;
    const long before = e == 0 ? prev : id[e - 1];
    first[e] = i == 0 || (a.by_change ? id[e] != before : before == a.eod);
    plain[e] = !(i < len && mark[e]);
  }
}

__global__ void __launch_bounds__(kThreads) document_plan_kernel(const Args a) {
  __shared__ Agg s_warp[32];
  __shared__ Agg s_step[kMaxSteps];  // reduction of every step of this CTA's chunk
  __shared__ Agg s_cta;              // reduction of the chunk (read by the other CTAs of the cluster)
  const int n_cta = (a.S + a.chunk - 1) / a.chunk;
  const int b = blockIdx.x / n_cta, rank = blockIdx.x % n_cta;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int c0 = rank * a.chunk, c1 = min(c0 + a.chunk, a.n_t * 128);
  const int n_steps = (c1 - c0 + kStep - 1) / kStep;
  pdl_trigger();
  pdl_wait();
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;

  // ---- reduce the chunk, step by step (a row of one step has nothing to carry over)
  const bool alone = n_cta == 1 && n_steps == 1;
  bool first[kPer], plain[kPer];  // of the last step read
  for (int st = 0; !alone && st < n_steps; ++st) {
    const int i0 = c0 + st * kStep + tid * kPer;
    load_flags(a, b, i0, len, first, plain);
    Agg g{-1, -1, a.S, a.S};
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i = i0 + e;
      if (i >= a.S) continue;
      if (first[e]) g.ds = i;
      if (first[e]) g.nf = min(g.nf, i);
      if (plain[e]) g.lu = i;
      if (first[e] || plain[e]) g.stop = min(g.stop, i);
    }
    g.ds = __reduce_max_sync(0xffffffffu, g.ds);
    g.lu = __reduce_max_sync(0xffffffffu, g.lu);
    g.stop = __reduce_min_sync(0xffffffffu, g.stop);
    g.nf = __reduce_min_sync(0xffffffffu, g.nf);
    if (lane == 0) s_warp[warp] = g;
    __syncthreads();
    if (warp == 0) {
      Agg w = s_warp[lane];
      w.ds = __reduce_max_sync(0xffffffffu, w.ds);
      w.lu = __reduce_max_sync(0xffffffffu, w.lu);
      w.stop = __reduce_min_sync(0xffffffffu, w.stop);
      w.nf = __reduce_min_sync(0xffffffffu, w.nf);
      if (lane == 0) {
        s_step[st] = w;
        if (st == 0) {
          s_cta = w;
        } else {
          s_cta.ds = max(s_cta.ds, w.ds);
          s_cta.lu = max(s_cta.lu, w.lu);
          s_cta.stop = min(s_cta.stop, w.stop);
          s_cta.nf = min(s_cta.nf, w.nf);
        }
      }
    }
    __syncthreads();
  }

  // ---- what lies left and right of this chunk
  Agg left{-1, -1, a.S, a.S}, right{-1, -1, a.S, a.S};
  if (n_cta > 1) {
    cluster_sync_all();
    Agg g{-1, -1, a.S, a.S};  // of CTA `lane`
    if (lane < n_cta)
      asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(g.ds), "=r"(g.lu), "=r"(g.stop), "=r"(g.nf)
                   : "r"(cluster_addr(&s_cta, lane))
                   : "memory");
    left.ds = __reduce_max_sync(0xffffffffu, lane < rank ? g.ds : -1);
    left.lu = __reduce_max_sync(0xffffffffu, lane < rank ? g.lu : -1);
    right.stop = __reduce_min_sync(0xffffffffu, lane > rank ? g.stop : a.S);
    right.nf = __reduce_min_sync(0xffffffffu, lane > rank ? g.nf : a.S);
  }

  // ---- scan and write, right to left
  int stop_right = right.stop, first_right = right.nf;
  for (int st = n_steps - 1; st >= 0; --st) {
    int ds_left = left.ds, lu_left = left.lu;
    for (int u = 0; u < st; ++u) {
      ds_left = max(ds_left, s_step[u].ds);
      lu_left = max(lu_left, s_step[u].lu);
    }
    const int i0 = c0 + st * kStep + tid * kPer;
    if (alone || st + 1 < n_steps) load_flags(a, b, i0, len, first, plain);
    int ds[kPer], lu[kPer], stop[kPer], nf[kPer];  // inclusive from the left / first stop and document start > i
    int rd = -1, rl = -1;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i = i0 + e;
      if (i < a.S && first[e]) rd = i;
      if (i < a.S && plain[e]) rl = i;
      ds[e] = rd;
      lu[e] = rl;
    }
    int rs = a.S, rf = a.S;
#pragma unroll
    for (int e = kPer - 1; e >= 0; --e) {
      stop[e] = rs;
      nf[e] = rf;
      if (i0 + e < a.S && first[e]) rf = i0 + e;
      if (i0 + e < a.S && (first[e] || plain[e])) rs = i0 + e;
    }
    const int sd = warp_max_scan(rd, lane), sl = warp_max_scan(rl, lane), ss = warp_min_scan_right(rs, lane),
              sf = warp_min_scan_right(rf, lane);
    __syncthreads();  // s_warp of the previous sweep has been read
    if (lane == 31) {
      s_warp[warp].ds = sd;
      s_warp[warp].lu = sl;
    }
    if (lane == 0) {
      s_warp[warp].stop = ss;
      s_warp[warp].nf = sf;
    }
    __syncthreads();
    int xd = ds_left, xl = lu_left, xs = stop_right, xf = first_right;
    {
      // the warps left of this one (starts, unmarked) and right of it (stops)
      const Agg w = s_warp[lane];
      xd = max(xd, __reduce_max_sync(0xffffffffu, lane < warp ? w.ds : -1));
      xl = max(xl, __reduce_max_sync(0xffffffffu, lane < warp ? w.lu : -1));
      xs = min(xs, __reduce_min_sync(0xffffffffu, lane > warp ? w.stop : a.S));
      xf = min(xf, __reduce_min_sync(0xffffffffu, lane > warp ? w.nf : a.S));
    }
    int pd = __shfl_up_sync(0xffffffffu, sd, 1), pl = __shfl_up_sync(0xffffffffu, sl, 1);
    int ns = __shfl_down_sync(0xffffffffu, ss, 1), nn = __shfl_down_sync(0xffffffffu, sf, 1);
    if (lane == 0) pd = pl = -1;
    if (lane == 31) ns = nn = a.S;
    xd = max(xd, pd);
    xl = max(xl, pl);
    xs = min(xs, ns);
    xf = min(xf, nn);
    if (!alone) {
      stop_right = min(stop_right, s_step[st].stop);
      first_right = min(first_right, s_step[st].nf);
    }

    int smin = INT_MAX, emax = 0, smax = 0, emin = INT_MAX;
    int qmin = INT_MAX, qemax = 0, qmax = 0, qemin = INT_MAX;
    int vs[kPer], ve[kPer], vp[kPer], ws[kPer], we[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i = i0 + e;
      vs[e] = ve[e] = vp[e] = ws[e] = we[e] = 0;
      if (i < len) {
        vs[e] = max(xd, ds[e]);
        const bool in_prefix = max(xl, lu[e]) < vs[e];
        ve[e] = in_prefix ? min(xs, stop[e]) : i + 1;
        ws[e] = in_prefix ? vs[e] : i;
        we[e] = min(min(xf, nf[e]), len);
        qmin = min(qmin, ws[e]);
        qemax = max(qemax, we[e]);
        vp[e] = i - vs[e];
        smin = min(smin, vs[e]);
        emax = max(emax, ve[e]);
      }
      if (i < a.S) {
        smax = max(smax, vs[e]);
        emin = min(emin, ve[e]);
        qmax = max(qmax, ws[e]);
        qemin = min(qemin, we[e]);
      }
    }
    const int tile = i0 / 128;  // one tile per warp
    if (tile < a.n_t) {
      const size_t row0 = (size_t)b * a.S;
      if (i0 + kPer <= a.S && (a.S & 3) == 0) {
        *reinterpret_cast<int4*>(a.positions + row0 + i0) = make_int4(vp[0], vp[1], vp[2], vp[3]);
        *reinterpret_cast<int4*>(a.start + row0 + i0) = make_int4(vs[0], vs[1], vs[2], vs[3]);
        *reinterpret_cast<int4*>(a.end + row0 + i0) = make_int4(ve[0], ve[1], ve[2], ve[3]);
      } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (i0 + e < a.S) {
            a.positions[row0 + i0 + e] = vp[e];
            a.start[row0 + i0 + e] = vs[e];
            a.end[row0 + i0 + e] = ve[e];
          }
      }
      int* tr = a.rows + ((size_t)b * a.n_t + tile) * 512 + lane * kPer;
      *reinterpret_cast<int4*>(tr) = make_int4(vs[0], vs[1], vs[2], vs[3]);
      *reinterpret_cast<int4*>(tr + 128) = make_int4(ve[0], ve[1], ve[2], ve[3]);
      *reinterpret_cast<int4*>(tr + 256) = make_int4(ws[0], ws[1], ws[2], ws[3]);
      *reinterpret_cast<int4*>(tr + 384) = make_int4(we[0], we[1], we[2], we[3]);
      smin = __reduce_min_sync(0xffffffffu, smin);
      emax = __reduce_max_sync(0xffffffffu, emax);
      smax = __reduce_max_sync(0xffffffffu, smax);
      emin = __reduce_min_sync(0xffffffffu, emin);
      qmin = __reduce_min_sync(0xffffffffu, qmin);
      qemax = __reduce_max_sync(0xffffffffu, qemax);
      qmax = __reduce_max_sync(0xffffffffu, qmax);
      qemin = __reduce_min_sync(0xffffffffu, qemin);
      if (lane == 0) {
        a.qstat[(size_t)b * a.n_t + tile] = make_int4(smin, emax, smax, emin);
        a.kstat[(size_t)b * a.n_t + tile] = make_int4(qmin, qemax, qmax, qemin);
      }
    }
  }
  if (n_cta > 1) cluster_sync_all();  // no CTA leaves while its s_cta may still be read
}

// Order in which the attention kernels take the tiles of all rows, heaviest first: a persistent grid hands tiles out
// in rounds, so the long ones have to come first and neighbours in a round be alike.  Counting sort by weight (key or
// query tiles to visit), one CTA for each of: pairs of query tiles, query tiles, key tiles.  The order of equals is
// left open; it changes when a tile is computed, not what is computed.
constexpr int kBins = 2048;
struct OrderArgs {
  const int4* qstat;
  const int4* kstat;
  int B, n_t, n_pairs, shift;  // weight >> shift < kBins
  int* out[3];
};

__device__ __forceinline__ int tile_weight(const int4* stat, const OrderArgs& a, int b, int t) {
  const int4 q = stat[(size_t)b * a.n_t + t];
  return q.y == 0 ? 0 : (q.y + 127) / 128 - q.x / 128;
}

__global__ void __launch_bounds__(kThreads) plan_order_kernel(const OrderArgs a) {
  __shared__ int s_bin[kBins];
  __shared__ int s_warp[32];
  const int which = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = which == 0 ? a.n_pairs : a.n_t;
  const int n = a.B * per;
  auto bin = [&](int e) {  // heaviest first
    const int b = e / per, t = e - b * per;
    int w;
    if (which == 0) {
      const int t1 = (a.n_t & 1) ? 2 * t : 2 * t + 1;
      w = tile_weight(a.qstat, a, b, t1) + (t1 > 0 ? tile_weight(a.qstat, a, b, t1 - 1) : 0);
    } else {
      w = tile_weight(which == 1 ? a.qstat : a.kstat, a, b, t);
    }
    return kBins - 1 - (w >> a.shift);
  };
  pdl_trigger();
  for (int k = tid; k < kBins; k += kThreads) s_bin[k] = 0;
  pdl_wait();
  __syncthreads();
  for (int e = tid; e < n; e += kThreads) atomicAdd(&s_bin[bin(e)], 1);
  __syncthreads();
  // exclusive scan over the bins, two to a thread
  const int c0 = s_bin[2 * tid], c1 = s_bin[2 * tid + 1];
  int v = c0 + c1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  const int base = v - c0 - c1 + (warp > 0 ? s_warp[warp - 1] : 0);
  s_bin[2 * tid] = base;
  s_bin[2 * tid + 1] = base + c0;
  __syncthreads();
  for (int e = tid; e < n; e += kThreads) a.out[which][atomicAdd(&s_bin[bin(e)], 1)] = e;
}
static_assert(kBins == 2 * kThreads, "two bins to a thread");

}  // namespace docplan

int document_plan_max_len() { return docplan::kMaxCtas * docplan::kMaxSteps * docplan::kStep; }

int document_plan(const long* ids, long ld_ids, long eod, int by_change, const unsigned char* marks, long ld_marks,
                  const int* lengths, int B, int S, int* positions, int* start, int* end, int* rows, void* qstat,
                  void* kstat, int* order, cudaStream_t stream) {
  using namespace docplan;
  if (B < 1 || S < 1 || S > document_plan_max_len() || (long)B * ((S + 127) / 128) > INT_MAX / 8) return -1;
  Args a;
  a.ids = ids;
  a.ld_ids = ld_ids;
  a.eod = eod;
  a.by_change = by_change;
  a.marks = marks;
  a.ld_marks = ld_marks;
  a.lengths = lengths;
  a.S = S;
  a.n_t = (S + 127) / 128;
  const int steps = (S + kStep - 1) / kStep;
  const int per_cta = (steps + kMaxCtas - 1) / kMaxCtas;
  a.chunk = per_cta * kStep;
  a.positions = positions;
  a.start = start;
  a.end = end;
  a.rows = rows;
  a.qstat = static_cast<int4*>(qstat);
  a.kstat = static_cast<int4*>(kstat);
  const int n_cta = (S + a.chunk - 1) / a.chunk;
  if ((long)B * n_cta > INT_MAX) return -2;
  const cudaError_t e = launch_early(n_cta, document_plan_kernel, (unsigned)(B * n_cta), kThreads, 0, stream, a);
  // rows of a few tiles: no tile is much heavier than another
  if (e != cudaSuccess || !order) return (int)e;
  OrderArgs o;
  o.qstat = a.qstat;
  o.kstat = a.kstat;
  o.B = B;
  o.n_t = a.n_t;
  o.n_pairs = (a.n_t + 1) / 2;
  o.shift = 0;
  while ((2 * a.n_t) >> o.shift >= kBins) ++o.shift;
  o.out[0] = order;
  o.out[1] = order + (size_t)B * o.n_pairs;
  o.out[2] = o.out[1] + (size_t)B * a.n_t;
  launch_early(0, plan_order_kernel, 3, kThreads, 0, stream, o);
  return (int)cudaGetLastError();
}

}  // namespace mmb
