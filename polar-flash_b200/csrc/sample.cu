// The draw of the next token (pf_sample_logits): temperature, top-k, top-p
// and min-p with a given uniform number, one thread-block cluster per row.
//
// With x_i = (l_i - max l) / T in 64 bits and w_i = exp(x_i) held as a whole
// number of 2^-44: sums of at most 2^19 such weights fit 64 bits and do not
// depend on their order, so atomics and any way to split a row give the same
// token.  The kept set of top-k and top-p is a prefix of the row sorted by
// (logit falling, index rising): all entries above some value, and the first
// few of those equal to it.  Neither needs a sort:
//   - the row is read once, a slice per CTA of the cluster, and stays in shared
//     memory (64 KB slices for vocabularies up to 131072);
//   - the value where the running count (top-k) or weight (top-p) from the top
//     reaches its target is found in a histogram of 2048 equal steps below the
//     maximum (logits spread over them, where their leading bits would crowd
//     into a few bins); what that step holds is compared all with all where it
//     is at most 256 entries, else put into histograms over its keys (fp32
//     bits as ordered integers) until one value is left;
//   - one warp of every CTA reads the others' sums of 64 bins each, then the 64
//     bins that matter, over distributed shared memory, and comes to the same
//     choice: one cluster barrier, and a twentieth of what reading every
//     histogram would move;
//   - the draw adds up weights by warp, finds the CTA, the warp's stretch and
//     the entry.
// Weights below 2^-45 of the largest are not computed.  A bin holds its weight
// in three 32-bit sums of 16-bit parts, which shared memory adds natively.
//
// 128256 fp32 logits, device time of 1 and 64 rows: greedy 8.8 and 24 us (the
// read, four barriers, two waves of CTAs), no filter 12 and 41 (an exponential
// each), top-k of 50 18 and 52, top-p of 0.9 37 and 119 (of it 13 and 39 the
// bins' atomics), all filters 26 and 71.  The read alone is 0.1 and 5 us: what
// bounds one row is its chain of passes and barriers, and many rows the same
// in two waves of CTAs: with top-p a warp spends a third of its time at
// barriers, 0.55 instructions are issued a cycle and scheduler, the FP64 pipe
// is busy 14 % of the time.
#include <cooperative_groups.h>
#include <math.h>

#include "common.cuh"
#include "launch.cuh"
#include "paged.cuh"

namespace cg = cooperative_groups;

namespace pfb {
namespace {

constexpr int kBins = 2048;
constexpr int kCand = 256;        // entries of a bin that are compared all with all
constexpr int kSlice = 16384;     // entries of a CTA, where eight CTAs suffice (64 KB: two CTAs an SM)
constexpr int kSmallSlice = 4096;
constexpr int kResident = 2 * 148;
constexpr int kMaxVocab = 360000;  // eight slices of 45000 (176 KB), each below 2^16 entries (bin sums)
constexpr int kMaxCluster = 8;
constexpr int kCta = 512;          // threads
typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  long long stride;
  int vocab, slice;  // slice: a multiple of 8
  const float *u, *ts, *ps, *ms;
  const int* ks;
  float t, p, m;
  int k;
  long long* tokens;
};

// Logits are kept as fp32 without NaN (which counts as -inf) and without -0, so
// that equal values have equal bits; their order as unsigned integers:
__device__ __forceinline__ float clean(float x) {
  if (x != x) x = -INFINITY;
  return x == 0.f ? 0.f : x;
}
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float of_key(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// What one CTA of the row's cluster knows.
struct Row {
  const float* v;  // its slice, -inf behind its end up to a multiple of 8
  int n;           // entries of it
  float top;       // the row's largest value
  double top_value, per_unit;  // log2(e) / T
  float bin_scale;             // steps of the first histogram per unit of logit

  // w = 2^y, y = (l - max l) log2(e) / T, off by at most 2^-46 of itself:
  // 2^n for the nearest integer n, times 2^f for |f| <= 1/2 by the polynomial
  // through 2^f at the Chebyshev points of degree 10 (3.2e-16).  0 below 2^-45.
  __device__ __forceinline__ double weight(float v) const {
    const double y = ((double)v - top_value) * per_unit;
    const bool low = !(y > -45.01);
    const double z = low ? 0.0 : y, big = z + 0x1.8p52, f = z - (big - 0x1.8p52);
    double p = 7.072585949269223e-09;
    p = fma(p, f, 1.0208690299958306e-07);
    p = fma(p, f, 1.321544258792169e-06);
    p = fma(p, f, 1.5252657260200837e-05);
    p = fma(p, f, 0.0001540353044173605);
    p = fma(p, f, 0.0013333558230164974);
    p = fma(p, f, 0.009618129107606888);
    p = fma(p, f, 0.05550410866444772);
    p = fma(p, f, 0.24022650695910097);
    p = fma(p, f, 0.69314718055995);
    p = fma(p, f, 1.0);
    p = __hiloint2double(__double2hiint(p) + (__double2loint(big) << 20), __double2loint(p));
    return v == top ? 1.0 : low ? 0.0 : p;
  }
  // w in units of 2^-44, rounded to the nearest (by an addition whose last bit is worth one).
  static __device__ __forceinline__ u64 whole(double w) {
    return (u64)__double_as_longlong(fma(w, 0x1p44, 0x1p52)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 fixed(float v) const { return whole(weight(v)); }
  // Steps below the maximum, the last one open; not falling as values fall.
  __device__ __forceinline__ float step(float v) const {
    return v == top ? 0.f : fminf((top - v) * bin_scale, (float)(kBins - 1));
  }
};

template <int kThreads>
struct alignas(16) Shared {
  static constexpr int kWarps = kThreads / 32;
  unsigned hist[4][kBins];  // weight in 16-bit parts (0, 1, 2), or entries (3); apart, so that a part's atomics spread over all banks
  u64 sums[kBins / 64];  // of 64 bins each
  float list[kCand];     // this CTA's entries of the chosen bin
  float all[kCand];      // the cluster's
  u64 all_mass[kCand];
  u64 pub_mass[2];
  int pub_count[2];
  float pub_lo[2], pub_hi[2];
  u64 warp_mass[kWarps];
  int warp_count[kWarps];
  float warp_lo[kWarps], warp_hi[kWarps];
  u64 sel_before, sel_held, sel_all;
  float sel_value, got_lo, got_hi;
  int lists[kMaxCluster];
  u64 got_total, got_mine;
  long long got_ties;
  int sel_bin, listed;
};

template <int kThreads>
struct Sampler {
  static constexpr int kWarps = kThreads / 32;
  using Sh = Shared<kThreads>;
  Sh& sh;
  Row row;
  int ranks, rank;
  // Parity of the pub_* that others may still read.  The histogram, its sums and
  // the list need no second copy: between the last look that another CTA takes
  // at one and its next change lies a cluster barrier.
  int turn = 0;

  __device__ __forceinline__ Sh& of(int r) { return ranks == 1 ? sh : *cg::this_cluster().map_shared_rank(&sh, r); }
  __device__ __forceinline__ void sync() {
    if (ranks == 1)
      __syncthreads();
    else
      cg::this_cluster().sync();
  }
  // f(x[4]) for the slice's values, in no order; the last ones may be -inf that is not of the slice.
  template <typename F>
  __device__ __forceinline__ void each4(F f) const {
    for (int i = 4 * threadIdx.x; i < row.n; i += 4 * kThreads) {
      const float4 q = *reinterpret_cast<const float4*>(row.v + i);
      const float x[4] = {q.x, q.y, q.z, q.w};
      f(x);
    }
  }

  static __device__ __forceinline__ float warp_min(float x) { return of_key(__reduce_min_sync(0xffffffffu, key_of(x))); }
  static __device__ __forceinline__ float warp_max(float x) { return of_key(__reduce_max_sync(0xffffffffu, key_of(x))); }

  // The cluster's smallest lo and largest hi; publishes `listed` beside them
  // (lane r of every warp receives CTA r's number of them).
  __device__ int min_max(float& lo, float& hi) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    lo = warp_min(lo);
    hi = warp_max(hi);
    if (lane == 0) {
      sh.warp_lo[warp] = lo;
      sh.warp_hi[warp] = hi;
    }
    __syncthreads();
    if (warp == 0) {
      lo = warp_min(lane < kWarps ? sh.warp_lo[lane] : INFINITY);
      hi = warp_max(lane < kWarps ? sh.warp_hi[lane] : -INFINITY);
      if (lane == 0) {
        sh.pub_lo[turn] = lo;
        sh.pub_hi[turn] = hi;
        sh.pub_count[turn] = sh.listed;
      }
    }
    sync();
    if (warp == 0) {  // a lane per CTA
      lo = warp_min(lane < ranks ? of(lane).pub_lo[turn] : INFINITY);
      hi = warp_max(lane < ranks ? of(lane).pub_hi[turn] : -INFINITY);
      if (lane < ranks) sh.lists[lane] = of(lane).pub_count[turn];
      if (lane == 0) {
        sh.got_lo = lo;
        sh.got_hi = hi;
      }
    }
    __syncthreads();
    lo = sh.got_lo;
    hi = sh.got_hi;
    turn ^= 1;
    return lane < ranks ? sh.lists[lane] : 0;
  }

  // Sums of 64 bins each, for the others to read behind the next barrier.
  // What bins b and b + 1 (b even) of a histogram hold.
  template <bool MASS>
  static __device__ __forceinline__ void held_by(const Sh& sh, int b, u64 (&m)[2]) {
    const uint2 x = *reinterpret_cast<const uint2*>(&sh.hist[MASS ? 0 : 3][b]);
    m[0] = x.x;
    m[1] = x.y;
    if (MASS) {
      const uint2 y = *reinterpret_cast<const uint2*>(&sh.hist[1][b]), z = *reinterpret_cast<const uint2*>(&sh.hist[2][b]);
      m[0] += ((u64)y.x << 16) + ((u64)z.x << 32);
      m[1] += ((u64)y.y << 16) + ((u64)z.y << 32);
    }
  }
  template <bool MASS>
  __device__ void add_bins() {
    const int lane = threadIdx.x & 31;
    __syncthreads();
    for (int g = threadIdx.x >> 5; g < kBins / 64; g += kWarps) {
      u64 h[2];
      held_by<MASS>(sh, 64 * g + 2 * lane, h);
      u64 m = h[0] + h[1];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      if (lane == 0) sh.sums[g] = m;
    }
  }

  // The first of the warp's lanes, in order, with which the running sum reaches
  // `target` (m: a lane's part, `run`: the sum before the warp's): (the lane, the
  // sum before it).  Where none reaches it, the last one that holds anything.
  static __device__ __forceinline__ int reach(u64 m, u64& run, double target) {
    const int lane = threadIdx.x & 31;
    u64 incl = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    incl += run;
    const unsigned some = __ballot_sync(0xffffffffu, m > 0), there = __ballot_sync(0xffffffffu, m > 0 && (double)incl >= target);
    const int at = there ? __ffs(there) - 1 : some ? 31 - __clz(some) : 0;
    run = __shfl_sync(0xffffffffu, incl - m, at);
    return at;
  }

  // Over the histograms of the cluster (behind add_bins and a barrier), the first
  // bin, from bin 0 up, with which the running sum reaches `target`, or, where
  // `share`, `target` times the sum of all: sh.sel_* receive it, what it holds and
  // the sum of the bins before it.  (The last one that holds anything where
  // none reaches it.)  MASS: weights; else entries.  Returns the sum of all.
  template <bool MASS>
  __device__ u64 choose(double target, bool share) {
    const int lane = threadIdx.x & 31;
    if (threadIdx.x < 32) {
      u64 v[kMaxCluster], m = 0;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) v[r] = r < ranks ? of(r).sums[lane] : 0;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) m += v[r];
      u64 all = m;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      if (share) target *= (double)all;
      u64 run = 0;
      const int g = reach(m, run, target);
      u64 h[2] = {0, 0}, q[kMaxCluster][2];  // bins 2 lane, 2 lane + 1 of the group
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
        if (r < ranks) held_by<MASS>(of(r), 64 * g + 2 * lane, q[r]);
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) h[i] += r < ranks ? q[r][i] : 0;
      const int at = reach(h[0] + h[1], run, target);
      const u64 a = __shfl_sync(0xffffffffu, h[0], at), b = __shfl_sync(0xffffffffu, h[1], at);
      // the first of the two, unless it holds nothing or only the second reaches the target
      const bool second = a == 0 || (b > 0 && !((double)(run + a) >= target));
      if (lane == 0) {
        sh.sel_bin = 64 * g + 2 * at + second;
        sh.sel_before = run + (second ? a : 0);
        sh.sel_held = second ? b : a;
        sh.sel_all = all;
      }
    }
    __syncthreads();
    return sh.sel_all;
  }

  // The value at which the running sum over the values from the top down reaches
  // `target` (MASS: that share of the whole weight, which `total` receives),
  // the sum of the values above it (`before`) and what equals it (`held`).
  // Entries below `floor` do not count; those equal to it weigh `floor_extra`
  // all together (MASS).
  template <bool MASS>
  __device__ float find(double target, float floor, u64 floor_extra, u64& before, u64& held, u64& total) {
    const int tid = threadIdx.x, lane = tid & 31;
    before = 0;
    float lo = floor, hi = row.top;
    for (int level = 0;; ++level) {
      for (int i = 4 * tid; i < kBins; i += 4 * kThreads)
#pragma unroll
        for (int part = MASS ? 0 : 3; part < (MASS ? 3 : 4); ++part)
          *reinterpret_cast<uint4*>(&sh.hist[part][i]) = make_uint4(0, 0, 0, 0);
      if (tid == 0) sh.listed = 0;
      __syncthreads();
      const unsigned khi = key_of(hi), span = khi - key_of(lo);
      const int shift = span >= kBins ? 32 - __clz(span / kBins) : 0;
      auto counts = [&](float v) { return v >= lo && v <= hi && v > -INFINITY; };
      auto bin_of = [&](float v) { return level == 0 ? (int)row.step(v) : (int)((khi - key_of(v)) >> shift); };
      unsigned tail = 0;
      each4([&](const float (&x)[4]) {
        if (!(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= lo)) return;
        if (MASS) {
          u64 w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = row.fixed(x[e]);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (counts(x[e]) && x[e] != floor && w[e]) {
              const int bin = bin_of(x[e]);
              const unsigned a = (unsigned)w[e] & 0xffffu, b = (unsigned)(w[e] >> 16) & 0xffffu, c = (unsigned)(w[e] >> 32);
              if (a) atomicAdd(&sh.hist[0][bin], a);
              if (b) atomicAdd(&sh.hist[1][bin], b);
              if (c) atomicAdd(&sh.hist[2][bin], c);
            }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool in = counts(x[e]);
            const int b = in ? bin_of(x[e]) : 0;
            const bool open = in && level == 0 && b == kBins - 1;  // can hold most of the row: not one by one
            tail += open;
            if (in && !open) atomicAdd(&sh.hist[3][b], 1u);
          }
        }
      });
      if (!MASS && level == 0) {
        tail = __reduce_add_sync(0xffffffffu, tail);
        if (lane == 0 && tail) atomicAdd(&sh.hist[3][kBins - 1], tail);
      }
      if (MASS && rank == 0 && tid == 0 && floor_extra && counts(floor)) {  // below 2^63
        const int bin = bin_of(floor);
        atomicAdd(&sh.hist[0][bin], (unsigned)floor_extra & 0xffffu);
        atomicAdd(&sh.hist[1][bin], (unsigned)(floor_extra >> 16) & 0xffffu);
        atomicAdd(&sh.hist[2][bin], (unsigned)(floor_extra >> 32));
      }
      add_bins<MASS>();
      sync();
      const u64 everything = choose<MASS>(level == 0 ? target : target - (double)before, MASS && level == 0);
      if (level == 0) {
        total = everything;
        if (MASS) target *= (double)everything;
      }
      const int b = sh.sel_bin;
      before += sh.sel_before;
      held = sh.sel_held;
      // the values that the bin holds: their ends, and the first of them as a list
      const float b_lo = (float)b, b_hi = (float)(b + 1);
      float vlo = INFINITY, vhi = -INFINITY;
      each4([&](const float (&x)[4]) {
        if (!(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= lo)) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          bool in = counts(x[e]);
          if (level == 0) {
            const float s = row.step(x[e]);
            in = in && s >= b_lo && s < b_hi;
          } else {
            in = in && (int)((khi - key_of(x[e])) >> shift) == b;
          }
          if (in) {
            vlo = fminf(vlo, x[e]);
            vhi = fmaxf(vhi, x[e]);
            const int i = atomicAdd(&sh.listed, 1);
            if (i < kCand) sh.list[i] = x[e];
          }
        }
      });
      const int n_of = min_max(vlo, vhi);
      lo = vlo;
      hi = vhi;
      if (lo >= hi) return hi;
      int upto = n_of;  // entries of the CTAs up to this lane's
#pragma unroll
      for (int o = 1; o < kMaxCluster; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      const int n = __shfl_sync(0xffffffffu, upto, ranks - 1);
      if (n > kCand || n < 0) continue;
      // few enough to compare all with all
      for (int r = 0; r < ranks; ++r) {
        const int end = __shfl_sync(0xffffffffu, upto, r), count = __shfl_sync(0xffffffffu, n_of, r);
        for (int i = tid; i < count; i += kThreads) {
          const float v = of(r).list[i];
          sh.all[end - count + i] = v;
          sh.all_mass[end - count + i] = !MASS ? 1 : v == floor ? 0 : row.fixed(v);
        }
      }
      __syncthreads();
      const double rest = target - (double)before;
      for (int i = tid; i < n; i += kThreads) {
        const float v = sh.all[i];
        u64 above = 0, equal = MASS && v == floor ? floor_extra : 0, sum = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
          const float u = sh.all[j];
          const u64 m = sh.all_mass[j];
          above += u > v ? m : 0;
          equal += u == v ? m : 0;
          sum += m;
        }
        if (MASS && lo == floor) sum += floor_extra;
        const bool never = !((double)sum >= rest);
        if (equal > 0 && (never ? above + equal == sum : ((double)above < rest || above == 0) && (double)(above + equal) >= rest)) {
          sh.sel_value = v;
          sh.sel_before = above;
          sh.sel_held = equal;
        }
      }
      __syncthreads();
      before += sh.sel_before;
      held = sh.sel_held;
      return sh.sel_value;
    }
  }

  // Weights above `cut` (of at least mp) and entries equal to it, by warp
  // (sh.warp_*: stretches of `per` entries, a multiple of 4) and published.
  __device__ void stretch_sums(float cut, double mp, int per) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int end = min(row.n, (warp + 1) * per);
    u64 mass = 0;
    unsigned count = 0;
    for (int base = warp * per; base < end; base += 128) {
      const int i = base + 4 * lane;
      const float4 q = i < end ? *reinterpret_cast<const float4*>(row.v + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      const float x[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) count += i + e < end && x[e] == cut;
      if (!__any_sync(0xffffffffu, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) > cut)) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const double w = row.weight(x[e]);
        mass += x[e] > cut && w >= mp ? Row::whole(w) : 0;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
    count = __reduce_add_sync(0xffffffffu, count);
    if (lane == 0) {
      sh.warp_mass[warp] = mass;
      sh.warp_count[warp] = (int)count;
    }
    __syncthreads();
    if (warp == 0) {
      mass = lane < kWarps ? sh.warp_mass[lane] : 0;
      count = __reduce_add_sync(0xffffffffu, lane < kWarps ? (unsigned)sh.warp_count[lane] : 0u);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
      if (lane == 0) {
        sh.pub_mass[turn] = mass;
        sh.pub_count[turn] = (int)count;
      }
    }
  }
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_kernel(const SampleArgs a) {
  constexpr int kWarps = kThreads / 32;
  extern __shared__ __align__(16) float vals[];
  __shared__ Shared<kThreads> sh;
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), r = blockIdx.x / ranks;
  const T* l = static_cast<const T*>(a.logits) + (long long)r * a.stride + (long long)rank * a.slice;
  const int n = max(0, min(a.slice, a.vocab - rank * a.slice));

  Sampler<kThreads> s{sh, Row{}, ranks, rank};
  // ---- the slice, and the row's largest value
  float lo = INFINITY, top = -INFINITY;
  constexpr int V = 16 / sizeof(T);
  const bool wide = (reinterpret_cast<uintptr_t>(l) & 15u) == 0;
  const int nv = wide ? n / V : 0;
#pragma unroll 4
  for (int i = tid; i < nv; i += kThreads) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(l) + i);
    T x[V];
    *reinterpret_cast<uint4*>(x) = q;
    float k[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      k[e] = clean(to_f32(x[e]));
      top = fmaxf(top, k[e]);
    }
#pragma unroll
    for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(vals + i * V + e) = make_float4(k[e], k[e + 1], k[e + 2], k[e + 3]);
  }
#pragma unroll 4
  for (int i = nv * V + tid; i < (n + 7) / 8 * 8; i += kThreads) {
    const float k = i < n ? clean(to_f32(l[i])) : -INFINITY;
    vals[i] = k;
    top = fmaxf(top, k);
  }
  const float tf = a.ts ? a.ts[r] : a.t, pf = a.ps ? a.ps[r] : a.p, mf = a.ms ? a.ms[r] : a.m, uf = a.u[r];
  const int k = a.ks ? a.ks[r] : a.k;
  if (tid == 0) sh.listed = 0;
  s.min_max(lo, top);
  if (top == -INFINITY) {  // the same in every CTA of the row
    if (rank == 0 && tid == 0) a.tokens[r] = -1;
    s.sync();
    return;
  }
  const bool greedy = !(tf > 0.f);
  s.row.v = vals;
  s.row.n = n;
  s.row.top = top;
  s.row.top_value = (double)top;
  const double t = greedy ? 1.0 : (double)tf;
  s.row.per_unit = 1.4426950408889634 / t;
  // the first histogram reaches 31.5 T below the maximum, where weights end
  s.row.bin_scale = (float)((double)(kBins - 1) / (31.5 * t));
  const double p = (double)pf, mp = fmin((double)mf, 1.0);

  // ---- kept: values > cut, and the first `ties` of those equal to it
  float cut = -INFINITY;
  long long ties = 0x7fffffff;
  if (greedy) {
    cut = top;
    ties = 1;
  } else {
    u64 before = 0, held = 0, total = 0;
    if (k > 0 && k < a.vocab) {
      cut = s.template find<false>((double)k, -INFINITY, 0, before, held, total);
      ties = (long long)k - (long long)before;
    }
    if (!(p >= 1.0)) {
      // what top-k keeps of the values at its cut weighs
      const u64 extra = (u64)min(ties, (long long)held) * s.row.fixed(cut);
      const float value = s.template find<true>(fmax(p, 0.0), cut, extra, before, held, total);
      const double want = p * (double)total;
      const u64 each = s.row.fixed(value);
      // entry j of the ties has before + j each in front of it: kept while that is less than want
      // (a quotient first, put right by the same comparison)
      auto kept = [&](long long j) { return (double)(before + (u64)j * each) < want; };
      long long a0 = a.vocab;
      if (each > 0) {
        a0 = (long long)fmin(fmax((want - (double)before) / (double)each, 0.0), (double)a.vocab);
        while (a0 > 0 && !kept(a0 - 1)) --a0;
        while (a0 < a.vocab && kept(a0)) ++a0;
      } else if (!kept(0)) {
        a0 = 0;
      }
      if (value == top) a0 = max(a0, 1ll);
      ties = value == cut ? min(ties, a0) : a0;
      cut = value;
    }
  }

  // ---- the draw: weights by stretch, in index order
  const int per = (n + 4 * kWarps - 1) / (4 * kWarps) * 4;
  s.stretch_sums(cut, mp, per);
  const u64 each = s.row.weight(cut) >= mp ? s.row.fixed(cut) : 0;  // (0 for -inf)
  s.sync();
  if (warp == 0) {
    // lane q holds CTA q's sums; kept ties are the first of all
    u64 q_mass = lane < ranks ? s.of(lane).pub_mass[s.turn] : 0;
    const long long q_ties = lane < ranks ? s.of(lane).pub_count[s.turn] : 0;
    long long tie_run = q_ties;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, tie_run, o);
      if (lane >= o) tie_run += y;
    }
    q_mass += (u64)max(0ll, min(q_ties, ties - (tie_run - q_ties))) * each;
    u64 mass_run = q_mass;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, mass_run, o);
      if (lane >= o) mass_run += y;
    }
    if (lane == ranks - 1) sh.got_total = mass_run;
    if (lane == rank) {  // kept weight and ties in front of this slice
      sh.got_mine = mass_run - q_mass;
      sh.got_ties = tie_run - q_ties;
    }
  }
  s.sync();  // the last look at another CTA's memory
  const u64 total = sh.got_total, mine = sh.got_mine;
  const long long my_ties = sh.got_ties;
  // running sum > u total, in whole numbers: > its floor; past the end (u >= 1), the last kept entry
  const double want = (double)uf * (double)total;
  const u64 w = want >= (double)total ? total - 1 : want > 0.0 ? (u64)want : 0;
  // the warp's stretch whose sums pass w
  u64 run = mine;
  long long seen = my_ties;
  int hit = -1;
  for (int q = 0; q < kWarps; ++q) {
    const long long c = sh.warp_count[q];
    const u64 next = run + sh.warp_mass[q] + (u64)max(0ll, min(c, ties - seen)) * each;
    if (run <= w && w < next) {
      hit = q;
      break;
    }
    run = next;
    seen += c;
  }
  if (hit < 0) return;  // not in this slice (block-uniform)
  // its entries, kThreads at a time
  __syncthreads();
  const int end = min(n, (hit + 1) * per);
  for (int base = hit * per; base < end; base += kThreads) {
    const int i = base + tid;
    const float v = i < end ? vals[i] : -INFINITY;
    const bool tie = i < end && v == cut;
    const unsigned vote = __ballot_sync(0xffffffffu, tie);
    u64 x = 0;
    if (v > cut) {
      const double e = s.row.weight(v);
      if (e >= mp) x = Row::whole(e);
    }
    // sums of the warp without ties first: a tie's rank needs the warps before
    if (lane == 0) sh.warp_count[warp] = __popc(vote);
    __syncthreads();
    long long rank_in = seen + __popc(vote & ((1u << lane) - 1u));
    int all = 0;
    for (int q = 0; q < kWarps; ++q) {
      if (q < warp) rank_in += sh.warp_count[q];
      all += sh.warp_count[q];
    }
    if (tie && rank_in < ties) x = each;
    u64 incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) sh.warp_mass[warp] = incl;
    __syncthreads();
    u64 sum = 0;
    for (int q = 0; q < kWarps; ++q) {
      if (q < warp) incl += sh.warp_mass[q];
      sum += sh.warp_mass[q];
    }
    incl += run;
    if (incl - x <= w && w < incl) a.tokens[r] = (long long)rank * a.slice + i;
    run += sum;
    seen += all;
    if (run > w) return;  // block-uniform
    __syncthreads();
  }
}

template <typename T, int kThreads>
cudaError_t launch_sample(const SampleArgs& a, int rows, int ranks, cudaStream_t st) {
  constexpr auto kern = sample_kernel<T, kThreads>;
  cudaError_t e = allow_smem<kern>(kMaxVocab / kMaxCluster * sizeof(float));
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)ranks, 1, 1};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)a.slice * sizeof(float);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, kern, a);
  note_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T>
cudaError_t launch_sample(SampleArgs a, int rows, cudaStream_t st) {
  int ranks = 1;
  while (ranks < kMaxCluster && (a.vocab + ranks - 1) / ranks > kSlice) ranks *= 2;
  // smaller slices while all CTAs still fit the machine at once: 1 row of 32001 with top-p 26.7 -> 20.8 us with
  // four CTAs for two, 32 rows 32.3 -> 29.7 us, but 256 rows 85 -> 114 us
  while (ranks < kMaxCluster && a.vocab / ranks > kSmallSlice && (long long)rows * ranks * 2 <= kResident) ranks *= 2;
  a.slice = ((a.vocab + ranks - 1) / ranks + 7) / 8 * 8;
  return launch_sample<T, kCta>(a, rows, ranks, st);
}

}  // namespace
}  // namespace pfb

using namespace pfb;

int pf_sample_logits(const void* logits, long long row_stride, int dtype, int rows, int vocab, const float* u,
                     const float* temperatures, float temperature, const int* top_ks, int top_k, const float* top_ps,
                     float top_p, const float* min_ps, float min_p, long long* tokens, void* stream) {
  if (!logits || !u || !tokens || rows < 0 ||
      (dtype != PF_DTYPE_F32 && dtype != PF_DTYPE_F16 && dtype != PF_DTYPE_BF16))
    return PF_ERR_INVALID_ARGUMENT;
  if (vocab <= 0 || vocab > kMaxVocab || row_stride < vocab) return PF_ERR_SHAPE;
  const uintptr_t size = dtype == PF_DTYPE_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(logits) % size) || !al4(u) || !al4(temperatures) || !al4(top_ks) || !al4(top_ps) ||
      !al4(min_ps) || (reinterpret_cast<uintptr_t>(tokens) & 7u))
    return PF_ERR_ALIGNMENT;
  if (rows == 0) return PF_OK;
  if (rows > 0x7fffffff / kMaxCluster) return PF_ERR_SHAPE;
  const SampleArgs a{logits, row_stride, vocab, 0, u, temperatures, top_ps, min_ps, top_ks, temperature, top_p, min_p,
                     top_k, tokens};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == PF_DTYPE_F32   ? launch_sample<float>(a, rows, s)
                        : dtype == PF_DTYPE_F16 ? launch_sample<__half>(a, rows, s)
                                                : launch_sample<__nv_bfloat16>(a, rows, s);
  return e == cudaSuccess ? PF_OK : report_cuda(e);
}
