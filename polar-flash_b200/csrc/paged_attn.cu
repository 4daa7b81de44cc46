// Attention of one new token per sequence over a paged KV cache
// (pf_paged_attention): out = sum_j p_j v_j / sum_j p_j, p_j = 2^(s_j - m),
// s_j = scale log2(e) q . k_j, m a running maximum.
//
// What it has to do is read the cache once, so everything is built around
// keeping reads in flight: each warp streams tiles of 16 positions (U of them
// per stage) of one (sequence, KV head) through its own cp.async ring in
// shared memory, and the warp alone waits for them.  Work is split over the
// length: the steps of all rows (sequence, KV head, group of eight query
// heads) lie in one order, kSetup units in front of each row for what starting
// it costs, and each CTA takes an equal run of that, whatever the lengths are.  A
// part of a row leaves (m, l, o) in the workspace and a second kernel joins the
// parts; sums are ordered, so results repeat.
//
// The products of the group's query heads with a tile are mma.sync (m16n8k16;
// 16 positions x 8 columns is what a tile has to offer, far below a tcgen05
// tile's 128 rows, and the reads are the bound):
//   S^T[16 positions][8] = K[16][hd] . Q^T,  O^T[hd][8] += V^T[hd][16] . W.
// Codes become exact fp16 values in registers (0x6400 | u is 1024 + u: a byte's
// u moved there, a 2-bit code where it stands in its 16-bit half, as c 2^b,
// the power of two going to q's and o's side), bf16 and fp16 rows are used as
// they are.  The fp32 operands on the other side keep their
// precision as sums of 16-bit terms: two fp16 ones, scaled by powers of two to
// just below fp16's largest value, so that what is a 2^-17th of the largest
// still has 22 bits, or three bf16 ones.  (q beside 2-bit codes stays below
// 2^13, and a 2^-8th of the largest has 22 bits wherever its code stands.)  Up to
// four query heads per KV head share the eight columns between two terms, more
// take a product per term; more than eight are units of their own, which read
// the row's cache again.
// A quantized row's value is s c + z (c a centred code), so  q . k = s_k (q . c) +
// z_k sum q  and  sum p v = sum (p s_v) c + sum p z_v: scales and zeros never
// touch the tiles.
// The maximum is taken of s_j + exponent(s_v), so the weights p s_v stay in
// range while rows differ in scale.
//
// Device time: 64 sequences of 300 to 4096 positions in bf16 pages, 32 heads
// over 8, 67 us (5.7 TB/s, 0.88 of the copy rate: bound by memory); the same in
// int8 58 us (3.5 TB/s); 8 of 9001 to 32768 in 2bit_asym, 64 heads over 8, 70 us
// (1.5 TB/s).  Quantized rows are bound by the instructions that turn codes into
// operands, 2 bits about 500 a tile in all, with two warps a scheduler that
// each issue one in 3.5 (2 bits) or 4.2 (int8) cycles.  One of 2048 in int8 takes
// 10.6 us (latency).  16-bit stages hold one tile of heads of 128 (8 KB), all
// others two.
#include <math.h>

#include "common.cuh"
#include "launch.cuh"
#include "paged.cuh"
#include "tma.cuh"

namespace pfb {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kHeads = 8;       // query heads of one unit
constexpr int kCtasPerSm = 2;
// steps that starting a row is worth (2, 4, 8: 64 sequences of 300 to 4096 in bf16 72.7, 67.2, 69.5 us;
// 8 of 9001 to 32768 in 2bit_asym 72.6, 70.4, 72.3)
constexpr int kSetup = 4;
constexpr int kRing = 25600;     // bytes of a warp's ring, at most

struct AttnArgs {
  KvPages pages;
  const void* q;
  void* out;
  const int *table, *lens;
  int dtype, width, seqs, nh, G, groups;
  float scale_log2;
  int2* parts;     // [seqs][nkv][groups]: first record, number of records (1: written to out)
  float* records;  // [2 CTAs][kHeads][hd + 2]: o (not yet divided), m, l
};

template <int MODE>
struct Mode {
  static constexpr bool kBf16 = MODE == PF_KV_BF16, k16 = kBf16 || MODE == PF_KV_F16;
  static constexpr bool k2 = MODE == PF_KV_2BIT || MODE == PF_KV_2BIT_ASYM, kAsym = MODE == PF_KV_2BIT_ASYM;
  static constexpr int kTerms = kBf16 ? 3 : 2;
  // log2 of the largest weight p.  Two fp16 terms want it high: p s_v stays below 2^15.  bf16 terms reach as far as
  // fp32, and so do bf16 values: sums over a million of the largest stay finite.
  static constexpr float kLift = kBf16 ? -20.f : 14.f;
};

template <int HD, int MODE, int PK>
struct Cfg {
  using M = Mode<MODE>;
  static constexpr int kNT = (M::kTerms + PK - 1) / PK;  // n tiles of 8 columns
  static constexpr int kRow = M::k16 ? 2 * HD : M::k2 ? HD / 4 : HD;
  static constexpr int kCpr = kRow / 16;                                 // 16-byte chunks of a row
  static constexpr int kU = M::k16 && HD == 128 ? 1 : 2;               // tiles of a stage (2-bit: 75.1 us with 4, 70.4 with 2)
  static constexpr int kJ = kU > 1 ? 2 : 1;  // tiles that go through the softmax together: fewer reductions, two chains at once
  static constexpr int kMeta = M::k16 ? 0 : M::kAsym ? 256 : 128;        // scales and zeros of a tile
  static constexpr int kTileBytes = 32 * kRow + kMeta;
  static constexpr int kStageBytes = kU * kTileBytes;
  static constexpr int kStages = kRing / kStageBytes < 6 ? kRing / kStageBytes : 6;
  static constexpr int kStep = kWarps * 16 * kU;  // positions of a CTA's step
  static constexpr int kKS = HD / 16, kMT = HD / 16;
  static constexpr int kQFrag = kNT * kKS * 32 * 8;
  static constexpr int kQRows = kHeads * HD * 4;
  static constexpr int kRings = kWarps * kStages * kStageBytes;
  // the rings also hold the warps' results after a run
  static constexpr int kMerge = kWarps * kHeads * (HD + 2) * 4;
  static constexpr size_t kSmem = kQFrag + kQRows + (kRings > kMerge ? kRings : kMerge);
  static_assert(kStages >= 2, "");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t b2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The maximum that a part of a row is joined by: maxima pass NaN scores over, the sum of weights does not.  A part
// of nothing but NaN would have the maximum -inf, and be left out as one without positions.
__device__ __forceinline__ float marked(float m, float l) { return l != l ? l : m; }
// Term `n` of x as a sum of 16-bit values, each the rounded rest of those before.
template <bool BF16>
__device__ __forceinline__ float term(float x, int n) {
  float t = 0.f;
  for (int i = 0; i <= n; ++i) {
    x -= t;
    t = BF16 ? __bfloat162float(__float2bfloat16_rn(x)) : __half2float(__float2half_rn(x));
  }
  return t;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  return BF16 ? b2(lo, hi) : h2(lo, hi);
}
template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// int8 codes (c + 128 in the bytes of u) as two fp16 pairs, exactly.
__device__ __forceinline__ uint32_t codes_lo(uint32_t u) {
  const uint32_t x = __byte_perm(u, 0x64646464u, 0x4140);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t u) {
  const uint32_t x = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 2-bit codes number i (0..7) of the two 16-bit halves of w (`low` = w << 2,
// `high` = w >> 6), as fp16 pairs (c - 1.5) 2^slot2(i), exactly.  (Centred, so
// that sums over many rows stay as small as the result; and not subnormals
// that would need no subtraction: the tensor cores align those by their
// written exponent and drop low bits.)
__host__ __device__ constexpr int slot2(int i) { return 2 + 2 * (i & 3); }
__device__ __forceinline__ uint32_t codes2(uint32_t low, uint32_t high, int i) {
  const uint32_t x = ((i < 4 ? low : high) & (0x00030003u << slot2(i))) | 0x64006400u;
  const __half2 off = __half2half2(__ushort_as_half((unsigned short)(0x6400 + (3 << slot2(i)) / 2)));  // 1024 + 1.5 2^slot2
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), off);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The place in its two bytes of code i: byte i / 4, value (3 - i % 4) of it.
__host__ __device__ constexpr int place2(int i) { return 4 * (i >> 2) + 3 - (i & 3); }

// The chunk where chunk c of tile row r is kept.  K is read by rows, eight
// lanes at a time over two rows (int8) or eight (ldmatrix); V by columns of
// chunks, over every second row.
template <int CPR, bool K16>
__device__ __forceinline__ int chunk_k(int r, int c) {
  if (K16) return c ^ (r & 7);
  return CPR == 8 ? c ^ ((r & 1) << 2) : c;
}
template <int CPR, bool K16>
__device__ __forceinline__ int chunk_v(int r, int c) {
  if (K16) return c ^ (r & 7);
  return CPR == 8 ? c ^ (r & 6) : CPR == 4 ? c ^ (r & 2) : c;
}

// The head dimension that k slot (ks, t, i) of the score products holds: slots
// 2t, 2t + 1 (i = 0, 1) and 2t + 8, 2t + 9 (i = 2, 3) of step ks, and, for
// 2-bit codes, the power of two (8 - slot2) that q is multiplied by there.
template <int HD, int MODE>
__device__ __forceinline__ int k_dim(int ks, int t, int i, int& shift) {
  using M = Mode<MODE>;
  shift = 0;
  if (M::k16) return 16 * ks + 2 * t + (i & 1) + 8 * (i >> 1);
  if (!M::k2) return 16 * (t + 4 * (ks >> 2)) + 4 * (ks & 3) + i;
  // word ks / 4 of the thread's HD / 64; codes 2 (ks % 4) and + 1 of its halves
  const int code = 2 * (ks & 3) + (i >> 1), byte = 4 * (ks >> 2) + 2 * (i & 1) + (code >> 2);
  shift = 8 - slot2(code);
  return 4 * ((HD / 16) * t + byte) + (place2(code) & 3);
}
// The head dimension of row g (which = 0) or g + 8 (1) of m tile mt of the
// value products, and the power of two its sums are multiplied by.
template <int HD, int MODE>
__device__ __forceinline__ int v_dim(int mt, int g, int which, int& shift) {
  using M = Mode<MODE>;
  shift = 0;
  if (M::k16) return 16 * mt + g + 8 * which;
  if (!M::k2) return (HD / 8) * g + 2 * mt + which;
  const int code = 2 * (mt & 3) + which;
  shift = slot2(code);
  return (HD / 8) * g + 8 * (mt >> 2) + 4 * (code >> 2) + (place2(code) & 3);
}

// Where the run of one of `ctas` CTAs starts, and the CTA that a unit belongs to
// (ctas <= units, so that no run is empty).
__device__ __forceinline__ long long run_start(long long units, int ctas, int cta) { return units * cta / ctas; }
__device__ __forceinline__ int run_of(long long units, int ctas, long long u) { return (int)(((u + 1) * ctas - 1) / units); }

template <int HD, int MODE, int PK>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_attn_kernel(const AttnArgs a) {
  using C = Cfg<HD, MODE, PK>;
  using M = Mode<MODE>;
  constexpr int NT = C::kNT, KS = C::kKS, MT = C::kMT, U = C::kU, S = C::kStages, J = C::kJ;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ long long warp_units[kWarps];
  __shared__ long long found_before;
  __shared__ int found_seq;
  __shared__ float head_mul[kHeads], head_sum[kHeads];
  __shared__ int valid_rows[kWarps][S][U];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint2* const qfrag = reinterpret_cast<uint2*>(smem);
  float* const qrow = reinterpret_cast<float*>(smem + C::kQFrag);  // [kHeads][HD], scaled
  unsigned char* const rings = smem + C::kQFrag + C::kQRows;
  pdl_enter();

  // ---- this CTA's run of units: seqs x nkv x groups x (kSetup + steps), in that order.
  // Thread i sums the units of a stretch of sequences; the one whose stretch
  // holds the run's start looks for its sequence.
  const int shift = a.pages.page_shift, nkv = a.pages.nkv, rows = nkv * a.groups;
  const long long cap = (long long)a.width << shift;
  auto length = [&](int b) { return (int)min((long long)max(a.lens[b], 0), min(cap, 0x7ff00000LL)); };
  // units of a row: none where there is nothing to read
  auto units_of = [&](int n) { return n > 0 ? (n + C::kStep - 1) / C::kStep + kSetup : 0; };
  const int per = (a.seqs + kThreads - 1) / kThreads, b0 = min(a.seqs, tid * per), b1 = min(a.seqs, b0 + per);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += (long long)units_of(length(b)) * rows;
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) warp_units[warp] = incl;
  __syncthreads();
  long long units = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) incl += warp_units[w];
    units += warp_units[w];
  }
  const int ctas = (int)min((long long)gridDim.x, units);
  if ((int)blockIdx.x >= ctas) return;  // block-uniform
  const long long lo = run_start(units, ctas, blockIdx.x), hi = run_start(units, ctas, blockIdx.x + 1);
  if (incl - mine <= lo && lo < incl) {
    long long before = incl - mine;
    int b = b0;
    for (; b < b1 - 1; ++b) {
      const long long n = (long long)units_of(length(b)) * rows;
      if (lo < before + n) break;
      before += n;
    }
    found_seq = b;
    found_before = before;
  }
  __syncthreads();
  int b = found_seq;
  long long seq0 = found_before;  // the first unit of sequence b

  for (long long u = lo; u < hi;) {
    // ---- one row: units u .. its end or the run's
    int len = length(b), row_units = units_of(len);
    while (u >= seq0 + (long long)row_units * rows) {
      seq0 += (long long)row_units * rows;
      ++b;
      len = length(b);
      row_units = units_of(len);
    }
    const int r = (int)((u - seq0) / row_units), kvh = r / a.groups, grp = r - kvh * a.groups;
    const long long row0 = seq0 + (long long)r * row_units;
    const int steps = row_units - kSetup;
    const int s0 = max(0, (int)(u - row0) - kSetup), s1 = (int)min((long long)row_units, hi - row0) - kSetup;
    u = row0 + row_units;
    if (s1 <= s0) continue;  // of this row, only what stands for its start
    const int heads = min(kHeads, a.G - grp * kHeads), h0 = kvh * a.G + grp * kHeads;

    // ---- the ring: the warp's tiles of step s are positions (s kWarps + warp) 16 U ..
    unsigned char* const ring = rings + warp * (S * C::kStageBytes);
    const uint32_t ring_s = smem_u32(ring);
    const int* const tab = a.table + (size_t)b * a.width;
    int next_page[U];
    auto look = [&](int s) {  // pages of step s, a step ahead of their use
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int p = ((s * kWarps + warp) * U + x) * 16;
        next_page[x] = s < s1 && p < len ? tab[p >> shift] : -1;
      }
    };
    auto load = [&](int s, int slot) {
#pragma unroll
      for (int x = 0; x < U; ++x) {
        const int p = ((s * kWarps + warp) * U + x) * 16, page = next_page[x];
        const bool ok = (unsigned)page < (unsigned)a.pages.num_pages;
        const int n = ok ? min(16, len - p) : 0;  // rows to read; the others become zeros
        if (lane == 0) valid_rows[warp][slot][x] = n;
        if (n > 0) {
          const size_t row = ((((size_t)page * nkv + kvh) << shift) + (p & ((1 << shift) - 1)));
          const unsigned char* const ks = static_cast<const unsigned char*>(a.pages.k) + row * C::kRow;
          const unsigned char* const vs = static_cast<const unsigned char*>(a.pages.v) + row * C::kRow;
          const uint32_t dk = ring_s + slot * C::kStageBytes + x * C::kTileBytes, dv = dk + 16 * C::kRow;
#pragma unroll
          for (int i = 0; i < (16 * C::kCpr + 31) / 32; ++i) {
            const int c = lane + 32 * i, rr = c / C::kCpr, cc = c % C::kCpr;
            if (16 * C::kCpr >= 32 || lane < 16 * C::kCpr) {
              cp16(dk + (rr * C::kCpr + chunk_k<C::kCpr, M::k16>(rr, cc)) * 16, ks + (rr < n ? c * 16 : 0), rr < n);
              cp16(dv + (rr * C::kCpr + chunk_v<C::kCpr, M::k16>(rr, cc)) * 16, vs + (rr < n ? c * 16 : 0), rr < n);
            }
          }
          if (!M::k16 && lane < C::kMeta / 16) {  // k scales, v scales, k zeros, v zeros: 64 bytes each
            const float* src = lane < 4 ? a.pages.k_scales : lane < 8 ? a.pages.v_scales : lane < 12 ? a.pages.k_zeros : a.pages.v_zeros;
            cp16(dk + 32 * C::kRow + lane * 16, src + row + 4 * (lane & 3), true);
          }
        } else if (M::k16 && C::kJ > 1) {
          // the other tile of its pair may be used: this one's values must be finite
          const uint32_t dv = ring_s + slot * C::kStageBytes + x * C::kTileBytes + 16 * C::kRow;
#pragma unroll
          for (int i = 0; i < 16 * C::kCpr / 32; ++i) cp16(dv + (lane + 32 * i) * 16, a.pages.v, false);
        }
      }
      cp_commit();
    };

    // ---- the first tiles and the group's query rows, asked for together
    float x[kHeads / kWarps][HD / 32];
#pragma unroll
    for (int k = 0; k < kHeads / kWarps; ++k)
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const int h = warp + k * kWarps;
        x[k][i] = h < heads ? load_x(a.q, a.dtype, ((size_t)b * a.nh + h0 + h) * HD + lane + 32 * i) : 0.f;
      }
    int first[S - 1][U];
#pragma unroll
    for (int i = 0; i < S - 1; ++i) {
      look(s0 + i);
#pragma unroll
      for (int k = 0; k < U; ++k) first[i][k] = next_page[k];
    }
    __syncthreads();  // the rings and fragments of the row before are free
#pragma unroll
    for (int i = 0; i < S - 1; ++i) {
#pragma unroll
      for (int k = 0; k < U; ++k) next_page[k] = first[i][k];
      load(s0 + i, i);
    }
    look(s0 + S - 1);
    // ---- the query rows as fragments, while the tiles arrive
    {
#pragma unroll
      for (int k = 0; k < kHeads / kWarps; ++k) {
        const int h = warp + k * kWarps;
        float top = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
          top = fmaxf(top, fabsf(x[k][i]));
          sum += x[k][i];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        // 2^e with top 2^-e in [2^14, 2^15) (2-bit codes: [2^6, 2^7), q is multiplied by up to 2^6
        // there); 1 for bf16, whose terms reach as far as fp32
        int e = 0;
        if (!M::kBf16 && top > 0.f)
          e = max(min((int)(__float_as_uint(top) >> 23) - 127 - (M::k2 ? 6 : 14), 120), -120);
        const float down = __uint_as_float((unsigned)(127 - e) << 23);
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) qrow[h * HD + lane + 32 * i] = x[k][i] * down;
        if (lane == 0) {
          // 2-bit codes carry 2^slot2, q there 2^(8 - slot2)
          head_mul[h] = __uint_as_float((unsigned)(127 + e) << 23) * (M::k2 ? 0x1p-8f : 1.f) * a.scale_log2;
          head_sum[h] = sum * a.scale_log2;
        }
      }
      __syncthreads();
      for (int i = tid; i < NT * KS * 32; i += kThreads) {
        const int nt = i / (KS * 32), ks = i / 32 % KS, ln = i & 31, col = ln >> 2, tt = ln & 3;
        const int h = PK == 2 ? col & 3 : col, tm = PK == 2 ? 2 * nt + (col >> 2) : nt;
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          int sh;
          const int d = k_dim<HD, MODE>(ks, tt, e, sh);
          y[e] = tm < M::kTerms ? term<M::kBf16>(qrow[h * HD + d] * (float)(1 << sh), tm) : 0.f;
        }
        qfrag[i] = make_uint2(pack<M::kBf16>(y[0], y[1]), pack<M::kBf16>(y[2], y[3]));
      }
    }
    // heads of this thread's two columns
    float mul[2], qsum[2];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int h = PK == 2 ? 2 * (t & 1) + e : 2 * t + e;
      mul[e] = head_mul[h];
      qsum[e] = head_sum[h];
    }

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, zs[2] = {0.f, 0.f};
    float o[MT][NT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;

    int slot = 0;
    for (int s = s0; s < s1; ++s) {
      cp_wait<S - 2>();
      __syncwarp();
#pragma unroll
      for (int x = 0; x < U; x += J) {
        int n[J], some = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) some |= n[j] = valid_rows[warp][slot][x + j];
        if (some == 0) continue;  // warp-uniform
        // sc[j][i][e]: tile j, position g + 8 i, column e
        float sc[J][2][2], up[J][2], vsc[J][2], vz[J][2];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          up[j][0] = up[j][1] = vz[j][0] = vz[j][1] = 0.f;
          vsc[j][0] = vsc[j][1] = 1.f;
          const unsigned char* const kt = ring + slot * C::kStageBytes + (x + j) * C::kTileBytes;
          const unsigned char* const vt = kt + 16 * C::kRow;
          const uint32_t kt_s = smem_u32(kt);
          // scores: rows g and g + 8
          float d[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[nt][e] = 0.f;
          auto score = [&](int ks, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint2 q = qfrag[(nt * KS + ks) * 32 + lane];
              mma<M::kBf16>(d[nt], a0, a1, a2, a3, q.x, q.y);
            }
          };
          if constexpr (M::k16) {
            const int rr = (lane & 7) + 8 * ((lane >> 3) & 1);  // matrices: rows 0-7, 8-15, then the next chunk
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              uint32_t f[4];
              ldsm4(kt_s + (rr * C::kCpr + chunk_k<C::kCpr, true>(rr, 2 * ks + (lane >> 4))) * 16, f);
              score(ks, f[0], f[1], f[2], f[3]);
            }
          } else if constexpr (!M::k2) {
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
              const uint4 x0 = *reinterpret_cast<const uint4*>(kt + (g * C::kCpr + chunk_k<C::kCpr, false>(g, t + 4 * c)) * 16);
              const uint4 x1 = *reinterpret_cast<const uint4*>(kt + ((g + 8) * C::kCpr + chunk_k<C::kCpr, false>(g + 8, t + 4 * c)) * 16);
              const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t y0 = w0[k] ^ 0x80808080u, y1 = w1[k] ^ 0x80808080u;
                score(4 * c + k, codes_lo(y0), codes_lo(y1), codes_hi(y0), codes_hi(y1));
              }
            }
          } else {
            uint32_t w0[HD / 64], w1[HD / 64];
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
              w0[c] = reinterpret_cast<const uint32_t*>(kt + g * C::kRow)[t * (HD / 64) + c];
              w1[c] = reinterpret_cast<const uint32_t*>(kt + (g + 8) * C::kRow)[t * (HD / 64) + c];
            }
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
              const uint32_t x0 = w0[c] << 2, x1 = w1[c] << 2, y0 = w0[c] >> 6, y1 = w1[c] >> 6;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                score(4 * c + k, codes2(x0, y0, 2 * k), codes2(x1, y1, 2 * k), codes2(x0, y0, 2 * k + 1),
                      codes2(x1, y1, 2 * k + 1));
            }
          }
          const float* const meta = reinterpret_cast<const float*>(kt + 32 * C::kRow);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const bool in = g + 8 * i < n[j];
            float ksc = 1.f, kz = 0.f;
            if (!M::k16) {
              ksc = meta[g + 8 * i];
              vsc[j][i] = meta[16 + g + 8 * i];
              if (M::kAsym) {  // s c + z = s (c - 1.5) + (z + 1.5 s)
                kz = fmaf(1.5f, ksc, meta[32 + g + 8 * i]);
                vz[j][i] = fmaf(1.5f, vsc[j][i], meta[48 + g + 8 * i]);
              }
              // the exponent of a positive scale (of what the codes' middle stands for, where that is larger: p z has
              // to stay in range too); the quantizer's smallest is 1e-8, less (a row never written) only makes the
              // weight small
              const float size = M::kAsym ? fmaxf(vsc[j][i], fabsf(vz[j][i])) : vsc[j][i];
              up[j][i] = (float)max((int)(__float_as_uint(size) >> 23) - 127, -30);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float y = d[0][2 * i + e];
#pragma unroll
              for (int nt = 1; nt < NT; ++nt) y += d[nt][2 * i + e];
              if (PK == 2) y += __shfl_xor_sync(0xffffffffu, y, 2);
              y *= mul[e];
              if (!M::k16) y *= ksc;
              if (M::kAsym) y = fmaf(kz, qsum[e], y);
              sc[j][i][e] = in ? y : -INFINITY;
            }
            if (!in) vsc[j][i] = vz[j][i] = up[j][i] = 0.f;
          }
        }
        float mx[2], keep[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(sc[0][0][e] + up[0][0], sc[0][1][e] + up[0][1]);
#pragma unroll
          for (int j = 1; j < J; ++j) mx[e] = fmaxf(mx[e], fmaxf(sc[j][0][e] + up[j][0], sc[j][1][e] + up[j][1]));
#pragma unroll
          for (int k = 4; k < 32; k <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], k));
          mx[e] = fmaxf(mx[e], m[e]);
          keep[e] = mx[e] == m[e] ? 1.f : ex2(m[e] - mx[e]);  // (0 from -inf)
        }
        if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            l[e] *= keep[e];
            zs[e] *= keep[e];
            m[e] = mx[e];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                o[i][nt][e] *= keep[e];
                o[i][nt][2 + e] *= keep[e];
              }
          }
        }
        float w[J][2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float top = (m[e] == -INFINITY ? 0.f : m[e]) - M::kLift;
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float p = ex2(sc[j][i][e] - top);  // 2^kLift times the weight: l and o alike
              l[e] += p;
              if (M::kAsym) zs[e] = fmaf(p, vz[j][i], zs[e]);
              w[j][i][e] = M::k16 ? p : p * vsc[j][i];
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const unsigned char* const kt = ring + slot * C::kStageBytes + (x + j) * C::kTileBytes;
          const unsigned char* const vt = kt + 16 * C::kRow;
          const uint32_t vt_s = smem_u32(vt);
          // weights [position][column] -> fragments [column][positions]
          uint32_t wf[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float y[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float first = term<M::kBf16>(w[j][i][e], 0);
                if (PK == 2) {  // terms 2 nt (lanes t < 2) and 2 nt + 1
                  if (nt == 0)
                    y[e] = t < 2 ? first : w[j][i][e] - first;
                  else
                    y[e] = t < 2 ? (w[j][i][e] - first) - term<M::kBf16>(w[j][i][e] - first, 0) : 0.f;
                } else {
                  y[e] = nt == 0 ? first : nt == 1 ? w[j][i][e] - first : (w[j][i][e] - first) - term<M::kBf16>(w[j][i][e] - first, 0);
                }
              }
              wf[nt][i] = transpose8(pack<M::kBf16>(y[0], y[1]));
            }
          auto value = [&](int mt, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<M::kBf16>(o[mt][nt], a0, a1, a2, a3, wf[nt][0], wf[nt][1]);
          };
          if constexpr (M::k16) {
            const int rr = (lane & 7) + 8 * (lane >> 4);  // matrices: chunk, the next one, then rows 8-15 of both
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t f[4];
              ldsm4t(vt_s + (rr * C::kCpr + chunk_v<C::kCpr, true>(rr, 2 * mt + ((lane >> 3) & 1))) * 16, f);
              value(mt, f[0], f[1], f[2], f[3]);
            }
          } else if constexpr (!M::k2) {
            // rows 2t, 2t + 1, 2t + 8, 2t + 9, the HD / 8 codes from g HD / 8
            uint32_t y[4][HD / 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int rr = 2 * t + (i & 1) + 8 * (i >> 1);
              if constexpr (HD == 128) {
                const uint4 f = *reinterpret_cast<const uint4*>(vt + (rr * C::kCpr + chunk_v<C::kCpr, false>(rr, g)) * 16);
                y[i][0] = f.x, y[i][1] = f.y, y[i][2] = f.z, y[i][3] = f.w;
              } else {
                const uint2 f = *reinterpret_cast<const uint2*>(vt + (rr * C::kCpr + chunk_v<C::kCpr, false>(rr, g >> 1)) * 16 + 8 * (g & 1));
                y[i][0] = f.x, y[i][1] = f.y;
              }
            }
#pragma unroll
            for (int k = 0; k < HD / 32; ++k) {
              const uint32_t p0 = __byte_perm(y[0][k], y[1][k], 0x5140) ^ 0x80808080u;
              const uint32_t p1 = __byte_perm(y[0][k], y[1][k], 0x7362) ^ 0x80808080u;
              const uint32_t q0 = __byte_perm(y[2][k], y[3][k], 0x5140) ^ 0x80808080u;
              const uint32_t q1 = __byte_perm(y[2][k], y[3][k], 0x7362) ^ 0x80808080u;
              value(2 * k, codes_lo(p0), codes_hi(p0), codes_lo(q0), codes_hi(q0));
              value(2 * k + 1, codes_lo(p1), codes_hi(p1), codes_lo(q1), codes_hi(q1));
            }
          } else {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const unsigned char* const p = vt + (2 * t + (i & 1) + 8 * (i >> 1)) * C::kRow + g * (HD / 32);
              y[i] = HD == 128 ? *reinterpret_cast<const uint32_t*>(p) : *reinterpret_cast<const uint16_t*>(p);
            }
#pragma unroll
            for (int hf = 0; hf < HD / 64; ++hf) {
              const uint32_t p = __byte_perm(y[0], y[1], hf ? 0x7632 : 0x5410);
              const uint32_t q = __byte_perm(y[2], y[3], hf ? 0x7632 : 0x5410);
              const uint32_t p0 = p << 2, p1 = p >> 6, q0 = q << 2, q1 = q >> 6;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                value(4 * hf + k, codes2(p0, p1, 2 * k), codes2(p0, p1, 2 * k + 1), codes2(q0, q1, 2 * k),
                      codes2(q0, q1, 2 * k + 1));
            }
          }
        }
      }
      __syncwarp();
      const int to = slot == 0 ? S - 1 : slot - 1;
      load(s + S - 1, to);
      look(s + S);
      slot = slot + 1 == S ? 0 : slot + 1;
    }
    cp_wait<0>();
    __syncthreads();  // the rings are free

    // ---- the warps' sums, side by side: [warp][head][HD] o, m, l
    float* const mg = reinterpret_cast<float*>(rings);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int k = 4; k < 32; k <<= 1) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], k);
        zs[e] += __shfl_xor_sync(0xffffffffu, zs[e], k);
      }
      const int h = PK == 2 ? 2 * (t & 1) + e : 2 * t + e;
      float* const rec = mg + (warp * kHeads + h) * (HD + 2);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float y = o[mt][0][2 * i + e];
#pragma unroll
          for (int nt = 1; nt < NT; ++nt) y += o[mt][nt][2 * i + e];
          if (PK == 2) y += __shfl_xor_sync(0xffffffffu, y, 2);
          int sh;
          const int dim = v_dim<HD, MODE>(mt, g, i, sh);
          if (PK == 1 || t < 2) rec[dim] = y * __uint_as_float((unsigned)(127 - sh) << 23) + zs[e];
        }
      if (g == 0 && (PK == 1 || t < 2)) {
        rec[HD] = marked(m[e], l[e]);
        rec[HD + 1] = l[e];
      }
    }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == steps;
    const int record = 2 * blockIdx.x + (s0 == 0);  // at most one part of each kind: the run's last row, and its first
    for (int h = warp; h < heads; h += kWarps) {
      float top = -INFINITY, wt[kWarps], ls = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, mg[(w * kHeads + h) * (HD + 2) + HD]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* rec = mg + (w * kHeads + h) * (HD + 2);
        wt[w] = rec[HD] == -INFINITY ? 0.f : ex2(rec[HD] - top);
        ls += wt[w] == 0.f ? 0.f : wt[w] * rec[HD + 1];
      }
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const int dim = lane + 32 * i;
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) y += wt[w] == 0.f ? 0.f : wt[w] * mg[(w * kHeads + h) * (HD + 2) + dim];
        if (whole) {
          store_as(a.out, a.dtype, ((size_t)b * a.nh + h0 + h) * HD + dim, ls == 0.f ? 0.f : y / ls);
        } else {
          a.records[((size_t)record * kHeads + h) * (HD + 2) + dim] = y;
        }
      }
      if (!whole && lane == 0) {
        a.records[((size_t)record * kHeads + h) * (HD + 2) + HD] = marked(top, ls);
        a.records[((size_t)record * kHeads + h) * (HD + 2) + HD + 1] = ls;
      }
    }
    if (tid == 0 && s0 == 0)  // the CTA of the first step describes the row's parts
      a.parts[((size_t)b * nkv + kvh) * a.groups + grp] =
          make_int2(record, run_of(units, ctas, row0 + row_units - 1) - (int)blockIdx.x + 1);
  }
}

// Joins a row's parts: the first CTA's record, then record 0 of the CTAs
// behind it.  A warp per query head; sequences without positions become zeros.
constexpr int kJoin = 16;  // parts in flight

template <int HD>
__global__ void __launch_bounds__(32 * kHeads) paged_join_kernel(const AttnArgs a) {
  const int lane = threadIdx.x & 31, h = threadIdx.x >> 5;
  pdl_enter();
  const int row = blockIdx.x, grp = row % a.groups, kvh = row / a.groups % a.pages.nkv, b = row / a.groups / a.pages.nkv;
  if (h >= a.G - grp * kHeads) return;
  const size_t at = ((size_t)b * a.nh + kvh * a.G + grp * kHeads + h) * HD;
  const int len = a.lens[b];
  const int2 p = a.parts[row];
  if (len <= 0) {
    for (int i = lane; i < HD; i += 32) store_as(a.out, a.dtype, at + i, 0.f);
    return;
  }
  if (p.y == 1) return;
  auto rec = [&](int i) {
    return a.records + ((size_t)(i == 0 ? p.x : 2 * (p.x / 2 + i)) * kHeads + h) * (HD + 2);
  };
  float top = -INFINITY, ls = 0.f, y[HD / 32];
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) y[i] = 0.f;
  for (int i0 = 0; i0 < p.y; i0 += kJoin) {  // a part's m and l per lane, its o by all lanes; asked for together
    const int n = min(kJoin, p.y - i0);
    float x[kJoin][HD / 32];
#pragma unroll
    for (int i = 0; i < kJoin; ++i)
#pragma unroll
      for (int k = 0; k < HD / 32; ++k) x[i][k] = i < n ? rec(i0 + i)[lane + 32 * k] : 0.f;
    const float m = lane < n ? rec(i0 + lane)[HD] : -INFINITY, l = lane < n ? rec(i0 + lane)[HD + 1] : 0.f;
    float mx = m;
#pragma unroll
    for (int o = kJoin / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mx = fmaxf(__shfl_sync(0xffffffffu, mx, 0), top);
    const float keep = top == mx ? 1.f : ex2(top - mx), w = m == -INFINITY ? 0.f : ex2(m - mx);
    float lw = w == 0.f ? 0.f : w * l;
#pragma unroll
    for (int o = kJoin / 2; o > 0; o >>= 1) lw += __shfl_xor_sync(0xffffffffu, lw, o);
    top = mx;
    ls = ls * keep + __shfl_sync(0xffffffffu, lw, 0);
#pragma unroll
    for (int k = 0; k < HD / 32; ++k) y[k] *= keep;
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
#pragma unroll
      for (int k = 0; k < HD / 32; ++k) y[k] += wi == 0.f ? 0.f : wi * x[i][k];
    }
  }
#pragma unroll
  for (int k = 0; k < HD / 32; ++k) store_as(a.out, a.dtype, at + lane + 32 * k, ls == 0.f ? 0.f : y[k] / ls);
}

// Streaming multiprocessors of the current device (cached per device).
int sm_count() {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev >= 0 && dev < 64 && cache[dev]) return cache[dev];
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev >= 0 && dev < 64) cache[dev] = n;
  return n;
}

size_t parts_bytes(int n_kv_heads, int groups, int seqs) {
  return ((size_t)seqs * n_kv_heads * groups * sizeof(int2) + 255) / 256 * 256;
}

template <int HD, int MODE, int PK>
cudaError_t launch_attn(const AttnArgs& a, int ctas, cudaStream_t s) {
  constexpr auto kern = paged_attn_kernel<HD, MODE, PK>;
  constexpr size_t smem = Cfg<HD, MODE, PK>::kSmem;
  const cudaError_t e = allow_smem<kern>(smem);
  if (e != cudaSuccess) return e;
  return launch_pdl_smem(kern, dim3(ctas), kThreads, smem, s, a);
}

template <int HD, int MODE>
cudaError_t launch_attn(const AttnArgs& a, int ctas, cudaStream_t s) {
  // up to four query heads: two terms of the fp32 operand share the eight columns
  return a.G <= 4 ? launch_attn<HD, MODE, 2>(a, ctas, s) : launch_attn<HD, MODE, 1>(a, ctas, s);
}

template <int HD>
cudaError_t launch_attn(const AttnArgs& a, int ctas, cudaStream_t s) {
  cudaError_t e;
  switch (a.pages.mode) {
    case PF_KV_INT8: e = launch_attn<HD, PF_KV_INT8>(a, ctas, s); break;
    case PF_KV_2BIT: e = launch_attn<HD, PF_KV_2BIT>(a, ctas, s); break;
    case PF_KV_2BIT_ASYM: e = launch_attn<HD, PF_KV_2BIT_ASYM>(a, ctas, s); break;
    case PF_KV_F16: e = launch_attn<HD, PF_KV_F16>(a, ctas, s); break;
    default: e = launch_attn<HD, PF_KV_BF16>(a, ctas, s);
  }
  if (e != cudaSuccess) return e;
  return launch_pdl(paged_join_kernel<HD>, dim3(a.seqs * a.pages.nkv * a.groups), 32 * kHeads, s, a);
}

}  // namespace
}  // namespace pfb

using namespace pfb;

size_t pf_paged_attention_workspace_size(int n_heads, int n_kv_heads, int head_dim, int seqs) {
  if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || head_dim <= 0 || seqs < 0) return 0;
  const int groups = (n_heads / n_kv_heads + kHeads - 1) / kHeads;
  // without a device (a query on the host alone) the count of a B200
  const int sms = sm_count() > 0 ? sm_count() : 148;
  return parts_bytes(n_kv_heads, groups, seqs) +
         (size_t)sms * kCtasPerSm * 2 * kHeads * (head_dim + 2) * sizeof(float);
}

int pf_paged_attention(const pf_kv_pages* pages, const void* q, int dtype, void* out, const int* block_table,
                       int table_width, const int* seq_lens, int seqs, int n_heads, float scale, void* workspace,
                       size_t workspace_bytes, void* stream) {
  const int st = pf_kv_pages_check(pages);
  if (st != PF_OK) return st;
  if (!q || !out || !block_table || !seq_lens || !workspace || seqs < 0 || !(fabsf(scale) <= 3e38f))
    return PF_ERR_INVALID_ARGUMENT;
  if (dtype != PF_DTYPE_F32 && dtype != PF_DTYPE_F16 && dtype != PF_DTYPE_BF16) return PF_ERR_INVALID_ARGUMENT;
  const int nkv = pages->n_kv_heads;
  if (n_heads <= 0 || n_heads % nkv || n_heads > 65535 || table_width <= 0 || (long long)seqs * n_heads > 0x7fffffffLL)
    return PF_ERR_SHAPE;
  if (!al16(q) || !al16(out) || !al16(workspace) || !al4(block_table) || !al4(seq_lens)) return PF_ERR_ALIGNMENT;
  if (workspace_bytes < pf_paged_attention_workspace_size(n_heads, nkv, pages->head_dim, seqs)) return PF_ERR_WORKSPACE;
  if (seqs == 0) return PF_OK;
  const int sms = sm_count();
  if (sms <= 0) return report_cuda(cudaErrorNoDevice);
  AttnArgs a{};
  a.pages = kv_pages(*pages);
  a.q = q;
  a.out = out;
  a.table = block_table;
  a.lens = seq_lens;
  a.dtype = dtype;
  a.width = table_width;
  a.seqs = seqs;
  a.nh = n_heads;
  a.G = n_heads / nkv;
  a.groups = (a.G + kHeads - 1) / kHeads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.parts = static_cast<int2*>(workspace);
  a.records = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + parts_bytes(nkv, a.groups, seqs));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = pages->head_dim == 128 ? launch_attn<128>(a, sms * kCtasPerSm, s)
                                               : launch_attn<64>(a, sms * kCtasPerSm, s);
  return e == cudaSuccess ? PF_OK : report_cuda(e);
}
