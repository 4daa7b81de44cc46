// Causal attention of packed prompts (pf_prompt_attention) on the
// 5th-generation tensor cores: O = softmax(scale Q K^T) V with a running row
// maximum m and sum l over key tiles,
//   p = 2^(c (s - m)),  c = scale log2 e,   l += sum p,   O += P V,
// where m only moves (and O and l are scaled by 2^(c (m_old - m_new))) when
// the row's maximum has grown by more than 2^8: until then p <= 2^8, which
// fp16 and bf16 hold as well as p <= 1, and the final O / l is the same.  For
// bf16, whose v may be near fp32's largest value, all p are lower by 2^20, so
// that sums over a million keys of it stay finite.
//
// The 128-row query tiles of one (sequence, KV head) are numbered
// x = (place in the prompt) * G + (query head in its group of G), and a CTA
// takes the tiles 2y and 2y + 1: for even G two heads at the same place, so
// both walk the same K and V tiles, each of which is loaded once for the two.
// CTAs of late places, which see the most keys, come first.
//
// Twelve warps, one CTA per SM:
//   warps 0-3, 4-7  softmax of tile 0 and 1, a thread per query row: S from
//             TMEM, mask, maximum, exponentials, P (16 bits) back into TMEM
//             over S; at the end O / l to global memory.
//   warp 8    TMA: Q once, then K and V tiles of 128 keys through a ring
//             (64-column boxes, 128B swizzle; columns past head_dim and rows
//             past the tensors arrive as zeros).
//   warp 9    tcgen05.mma from one lane: S = Q K^T (both from shared memory,
//             K-major), O += P V (P from TMEM, V from shared memory with its
//             head dimension contiguous).  While one tile's softmax runs, the
//             other tile's products do.  V rows behind the sequence's end are
//             zeroed before use: they belong to other sequences and may hold
//             anything, and 0 * NaN would reach O.
//   warps 10, 11  none: their registers go to the softmax.
// TMEM: S0 S1 (128 fp32 columns each; P over the first 64), O0 O1.
//
// One tile's chain of a step (heads of 128, in cycles): scores there to P handed
// over 1800 (reads 45, maximum 330, exponentials 1300, P 150), 100 until the
// products are issued, 1370 for P V and the next scores; the other tile's chain
// fills half of that.  The exponentials (16384 a tile, 16 a cycle and SM) are
// the longest part.  8192 tokens, 32 heads over 8, bf16: 440 us in a burst of
// three calls (1.25 PFLOP/s), 515 us sustained under the power limit.  Heads of
// 96 take the form of 128 (12 prompts to 1500 tokens, 52 and 51 us), 40 that of
// 64 (45 and 42): the softmax, which costs the same, bounds them.  Weights are
// rounded to 16 bits because that is what the products take beside a 16-bit v;
// it takes the normwise error in bf16 from the 1.6e-3 of the output's own
// rounding to 2.0e-3.
// Tried and slower.  Sustained, each beside the form of its day: two threads per
// row (595 against 545 us), three pairs of exponentials in eight on the FMA pipes
// instead of one (527 against 516).  In bursts, against 443 us: steps of 64 keys
// with two S buffers (558: 64-wide score products wait for Q's reads from shared
// memory), a warp of products per tile (534: their products interleave), and a
// warp that waits together and votes (457).
// Every wait is bounded.  One that gives up raises the CTA's abort flag, on
// which the other waits give up too; the status word is marked, and rows that
// were still waiting become NaN.  The warps then meet at a barrier, and only
// behind it, where nothing more is issued, the loading thread waits for every
// copy that it issued and the issuing thread for its products, before TMEM is
// freed and the block ends.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "paged.cuh"
#include "tma.cuh"

namespace pfb {
namespace {

constexpr int kTile = 128;  // query rows, and keys, of a tile
constexpr int kThreads = 384;
constexpr int kTmaWarp = 8, kMmaWarp = 9;
constexpr uint32_t kBox = kTile * 128;  // bytes of a 64-column box
constexpr int kTmemS = 0, kTmemO = 256, kTmemCols = 512;
constexpr float kSlack = 8.f;  // log2 of the largest p
template <typename T>
constexpr float kLower = std::is_same<T, __nv_bfloat16>::value ? 20.f : 0.f;  // p is 2^-kLower times the weight
constexpr int kPoly = 1;       // of eight pairs of exponentials, those on the FMA pipes

struct PromptArgs {
  const void *q, *k, *v;
  void* out;
  long long qs, ks, vs, os;
  const int *cu_q, *cu_k;
  int seqs, total_q, total_k, G, nkv, hd;
  float scale_log2;
  unsigned* status;
  unsigned poll_mask;          // of polls of a wait, those that look at the clock: every poll_mask + 1st
  unsigned long long wait_ns;  // after which a wait gives up
};

template <int HD>
struct Cfg {
  static constexpr int kBoxes = HD / 64;
  static constexpr uint32_t kTileBytes = kBoxes * kBox;
  static constexpr int kStages = HD == 128 ? 4 : 8;
  static constexpr size_t kSmem = (2 + kStages) * (size_t)kTileBytes + 1024;
};

// Bounded wait on an mbarrier phase, polling without a suspend hint and
// looking at the clock and the abort flag every 64th time only (both cost
// more than a poll, and the kernel's chain of waits is its critical path);
// false when it gave up or another warp of the CTA did.  The answer is the
// calling thread's own: a warp that goes on together takes a vote of it.
constexpr unsigned kPollMask = 63;
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const volatile int* abort_flag, unsigned mask,
                                         unsigned long long limit_ns) {
  unsigned long long t0 = 0;
  for (unsigned spin = 1;; ++spin) {
    uint32_t done;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if (spin & mask) continue;
    if (*abort_flag) return false;
    const unsigned long long t = now_ns();
    if (t0 == 0)
      t0 = t;
    else if (t - t0 >= limit_ns)
      return false;
  }
}

// One lane of a whole warp, always the same one; the branch on it is known to
// the compiler, which keeps the operands of the products in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{ .reg .pred P; elect.sync _|P, 0xffffffff; selp.u32 %0, 1, 0, P; }" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Shared-memory operand descriptors, 128B swizzle.  K-major (Q, K): 8-row
// groups 1024 bytes apart.  MN-major (V: keys are rows, head dimensions
// contiguous): groups of 8 keys 1024 bytes apart, 64-column boxes kBox apart.
__device__ __forceinline__ uint64_t desc_k(uint32_t a) {
  return (uint64_t)((a & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t a) {
  return (uint64_t)((a & 0x3FFFFu) >> 4) | ((uint64_t)(kBox >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// M = 128, N = n, fp32 D; fp16 or bf16 A and B; B MN-major where `mn`.
__host__ __device__ constexpr uint32_t idesc(bool bf16, int n, bool mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTile >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
               "l"(a), "l"(b), "r"(id), "r"(acc)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(
                   d),
               "r"(a), "l"(b), "r"(id), "r"(acc)
               : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define PF_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define PF_W8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : PF_R8(v, 0), PF_R8(v, 8), PF_R8(v, 16), PF_R8(v, 24)
      : "r"(a));
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::PF_W8(v, 0),
      PF_W8(v, 8), PF_W8(v, 16), PF_W8(v, 24), "r"(a)
      : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two fp32 values as the packed operations take them.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^x of two values on the FMA pipes: x = n + f with n the nearest integer
// (its bits taken from x + 1.5 2^23), 2^f for |f| <= 1/2 by the polynomial of
// least relative error (degree 3: 7.5e-5, a fiftieth of bf16's half step;
// degree 4: 2.6e-6, a two-hundredth of fp16's), n added to the exponent.
// x <= 127.  Masked and far lower scores end at kFloor, just above -127: there
// n = -127 takes the exponent of a polynomial a little above 1 to zero, and what
// is left, about 2^-139, is 0 in either type (2^-126 is a bf16 number, which a
// large v would show).  Between kFloor and -126 the weight falls from 2^-126
// to that.  NaN gives a number near fp32's largest or more, which the row's sum
// is looked at for.
constexpr float kFloor = -126.9998f;
template <typename T>
__device__ __forceinline__ void ex2_poly(uint64_t x, float& lo, float& hi) {
  f2_split(x, lo, hi);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(kFloor));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(kFloor));
  x = f2(lo, hi);
  const uint64_t t = add2(x, f2(12582912.f, 12582912.f));
  const uint64_t f = fma2(add2(t, f2(-12582912.f, -12582912.f)), f2(-1.f, -1.f), x);
  uint64_t p;
  if (std::is_same<T, __half>::value) {
    p = fma2(f2(0.009570102207362652f, 0.009570102207362652f), f, f2(0.05591785907745361f, 0.05591785907745361f));
    p = fma2(p, f, f2(0.240247443318367f, 0.240247443318367f));
    p = fma2(p, f, f2(0.6931217908859253f, 0.6931217908859253f));
    p = fma2(p, f, f2(0.9999992847442627f, 0.9999992847442627f));
  } else {
    p = fma2(f2(0.0551716685295105f, 0.0551716685295105f), f, f2(0.2426111251115799f, 0.2426111251115799f));
    p = fma2(p, f, f2(0.6932609677314758f, 0.6932609677314758f));
    p = fma2(p, f, f2(0.9999280571937561f, 0.9999280571937561f));
  }
  float tl, th;
  f2_split(t, tl, th);
  f2_split(p, lo, hi);
  lo = __uint_as_float(__float_as_uint(lo) + (__float_as_uint(tl) << 23));
  hi = __uint_as_float(__float_as_uint(hi) + (__float_as_uint(th) << 23));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// What waits that gave up left on a device (pf_prompt_status): in the library's
// own image, so that every call reports to it, captured ones too.
static __device__ unsigned g_prompt_status;

// What a CTA works on: sequence rows, and per tile its head, first row and
// number of key tiles.
struct Job {
  int q0, k0, n, m;  // first query and key row of the sequence, their numbers
  int kvh;
  int head[2], row0[2], tiles[2];  // head -1: no such tile
};

// The warp's job of block `idx`; false where there is none.  Every read of cu_q
// and cu_k stays inside them, and rows are limited to the tensors, whatever
// they hold.
__device__ __forceinline__ bool find_job(const PromptArgs& a, int idx, Job& job) {
  const int lane = threadIdx.x & 31;
  job.kvh = idx % a.nkv;
  int y = idx / a.nkv;
  for (int base = 0; base < a.seqs; base += 32) {
    const int b = base + lane;
    int q0 = 0, n = 0;
    if (b < a.seqs) {
      q0 = min(max(a.cu_q[b], 0), a.total_q);
      n = max(min(a.cu_q[b + 1], a.total_q) - q0, 0);
    }
    const int tiles = (n + kTile - 1) / kTile * a.G, pairs = (tiles + 1) / 2;
    int run = pairs;  // inclusive sum over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += t;
    }
    const unsigned past = __ballot_sync(0xffffffffu, run > y);
    if (past) {
      const int src = __ffs(past) - 1;
      const int before = __shfl_sync(0xffffffffu, run - pairs, src), all = __shfl_sync(0xffffffffu, pairs, src);
      const int total = __shfl_sync(0xffffffffu, tiles, src);
      job.q0 = __shfl_sync(0xffffffffu, q0, src);
      job.n = __shfl_sync(0xffffffffu, n, src);
      const int s = base + src;
      job.k0 = min(max(a.cu_k[s], 0), a.total_k);
      job.m = max(min(a.cu_k[s + 1], a.total_k) - job.k0, 0);
      const int pair = all - 1 - (y - before);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int x = 2 * pair + t;
        job.head[t] = x < total ? job.kvh * a.G + x % a.G : -1;
        job.row0[t] = x / a.G * kTile;
        // the last key that the tile's last row sees
        const int last = job.m - job.n + min(job.n - 1, job.row0[t] + kTile - 1);
        job.tiles[t] = x < total && last >= 0 ? last / kTile + 1 : 0;
      }
      return true;
    }
    y -= __shfl_sync(0xffffffffu, run, 31);
  }
  return false;
}

// A NaN or infinity in v at a key that a row does not see meets the weight 0 in
// the products of the row's last tile, and makes NaN of it.  For `kDims` output
// values of a row (from dim0) that came out not finite: whether one of the keys
// seen + 1 .. end - 1 has such a value there; then the values are computed
// again over the keys that the row sees, and stored.
constexpr int kDims = 32;
template <typename T>
__device__ __noinline__ bool without_hidden(const PromptArgs& a, int q_row, int head, int k0, int kvh, int seen, int end,
                                            int dim0, float mc, float inv) {
  const T* const q = static_cast<const T*>(a.q) + (long long)q_row * a.qs + (long long)head * a.hd;
  const T* const k = static_cast<const T*>(a.k) + (long long)k0 * a.ks + (long long)kvh * a.hd;
  const T* const v = static_cast<const T*>(a.v) + (long long)k0 * a.vs + (long long)kvh * a.hd + dim0;
  const int dims = min(kDims, a.hd - dim0);
  bool hidden = false;
  for (int j = seen + 1; j < end; ++j)
    for (int e = 0; e < dims; ++e) hidden = hidden || !isfinite(to_f32(v[j * a.vs + e]));
  if (!hidden) return false;
  float o[kDims];
  for (int e = 0; e < dims; ++e) o[e] = 0.f;
  for (int j = 0; j <= seen; ++j) {
    float x = 0.f;
    for (int d = 0; d < a.hd; ++d) x = fmaf(to_f32(q[d]), to_f32(k[j * a.ks + d]), x);
    const float p = to_f32(from_f32<T>(ex2(fmaf(x, a.scale_log2, -mc))));
    for (int e = 0; e < dims; ++e) o[e] = fmaf(p, to_f32(v[j * a.vs + e]), o[e]);
  }
  T* const out = static_cast<T*>(a.out) + (long long)q_row * a.os + (long long)head * a.hd + dim0;
  for (int e = 0; e < dims; ++e) out[e] = from_f32<T>(o[e] * inv);
  return true;
}

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PromptArgs a) {
  using C = Cfg<HD>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kStages = C::kStages;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ uint64_t bars[2 * kStages + 10];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int copies;  // ring entries whose copies were issued
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t full0 = smem_u32(&bars[0]), free0 = smem_u32(&bars[kStages]), qbar = smem_u32(&bars[2 * kStages]);
  const uint32_t sbar = qbar + 8, obar = qbar + 24, dbar = qbar + 40;  // s, o: one per tile
  const uint32_t pbar = qbar + 48;                                     // one per tile and half of P
  const uint32_t ring = base + 2 * C::kTileBytes;
  const volatile int* abort_p = &abort_flag;

  if (threadIdx.x == 0) {
    abort_flag = copies = 0;
    for (int s = 0; s < 2 * kStages + 10; ++s) {
      // p: the four softmax warps of a tile arrive
      const bool p = s >= 2 * kStages + 6;
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full0 + 8 * s), "r"(p ? 4 : 1));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_enter();
  auto wait = [&](uint32_t bar, uint32_t parity) { return bar_wait(bar, parity, abort_p, a.poll_mask, a.wait_ns); };
  Job job;
  if (find_job(a, blockIdx.x, job)) {
    const int most = max(job.tiles[0], job.tiles[1]);
    // 12 warps of 168 registers: the eight softmax warps take 208, the others
    // keep 88 (8 * 208 + 4 * 88 = 12 * 168)
    if (warp >= kTmaWarp) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if (warp == kTmaWarp) {
        // ---------------------------------------------------------- loads
        if (lane == 0 && most > 0) {
          const uint32_t nq = (job.tiles[0] > 0) + (job.tiles[1] > 0);
          mbar_expect(qbar, nq * C::kTileBytes);
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (job.tiles[t] > 0)
              for (int x = 0; x < C::kBoxes; ++x)
                tma_3d(base + t * C::kTileBytes + x * kBox, &qmap, 64 * x, job.head[t], job.q0 + job.row0[t], qbar);
          for (int i = 0; i < 2 * most; ++i) {  // K and V in turn
            const int slot = i % kStages;
            if (i >= kStages && !wait(free0 + 8 * slot, (i / kStages - 1) & 1)) {
              abort_flag = 1;
              break;
            }
            const uint32_t bar = full0 + 8 * slot, dst = ring + slot * C::kTileBytes;
            mbar_expect(bar, C::kTileBytes);
            for (int x = 0; x < C::kBoxes; ++x)
              tma_3d(dst + x * kBox, i & 1 ? &vmap : &kmap, 64 * x, job.kvh, job.k0 + (i >> 1) * kTile, bar);
            copies = i + 1;
          }
        }
      } else if (warp == kMmaWarp) {
        // ---------------------------------------------------------- products
        const uint32_t id_s = idesc(kBf16, kTile, false), id_o = idesc(kBf16, HD, true);
        auto score = [&](int t, int i) {  // S_t = Q_t K^T, K in ring entry i
          const uint32_t sa = base + t * C::kTileBytes, sb = ring + (i % kStages) * C::kTileBytes;
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {
            const uint32_t off = (k >> 2) * kBox + (k & 3) * 32;
            mma_ss(tmem + kTmemS + t * kTile, desc_k(sa + off), desc_k(sb + off), id_s, k > 0);
          }
          commit(sbar + 8 * t);
        };
        // The steps are one thread's: it waits and issues by itself (with a vote of the warp at each wait 8192 tokens
        // took 457 us for 445).  The warp meets before the last step, where a V tile that the sequence does not fill needs
        // zeros, and once more at the end; `ok` is the same in all lanes there.
        bool ok = true;
        for (int from = 0; ok && from < most;) {
          const int whole = job.m / kTile, to = from < whole && whole < most ? whole : most;
          const int last = 2 * to - 1, left = job.m - (to - 1) * kTile;  // V of the last step, keys of the sequence in it
          if (left < kTile) {
            const uint32_t sv = ring + (last % kStages) * C::kTileBytes;
            ok = __all_sync(0xffffffffu, wait(full0 + 8 * (last % kStages), (last / kStages) & 1));
            if (!ok) break;
            for (int r = left * 8 + lane; r < kTile * 8; r += 32)
              for (int x = 0; x < C::kBoxes; ++x)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sv + x * kBox + r * 16), "r"(0) : "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          if (elect_one()) {
            if (from == 0) {
              ok = wait(qbar, 0) && wait(full0, 0);
              if (ok) {
                fence_after();
#pragma unroll
                for (int t = 0; t < 2; ++t)
                  if (job.tiles[t] > 0) score(t, 0);
                commit(free0);
              }
            }
            for (int j = from; ok && j < to; ++j) {
              const int iv = 2 * j + 1, ik = 2 * j + 2;
              ok = wait(full0 + 8 * (iv % kStages), (iv / kStages) & 1);
              if (!ok) break;
              const uint32_t sv = ring + (iv % kStages) * C::kTileBytes;
              bool have_k = false;
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                if (!ok || j >= job.tiles[t]) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // P and the products with it in two halves of the keys
                  ok = ok && wait(pbar + 16 * t + 8 * h, j & 1);
                  if (!ok) continue;
                  fence_after();
#pragma unroll
                  for (int k = 4 * h; k < 4 * h + 4; ++k)
                    mma_ts(tmem + kTmemO + t * HD, tmem + kTmemS + t * kTile + 8 * k, desc_mn(sv + k * 2048), id_o,
                           j > 0 || k > 0);
                  if (h) commit(obar + 8 * t);
                }
                if (!ok) continue;
                if (j + 1 < job.tiles[t]) {
                  if (!have_k) ok = wait(full0 + 8 * (ik % kStages), (ik / kStages) & 1);
                  if (!ok) continue;
                  have_k = true;
                  fence_after();
                  score(t, ik);
                }
              }
              if (ok) {
                commit(free0 + 8 * (iv % kStages));
                if (j + 1 < most) commit(free0 + 8 * (ik % kStages));
              }
            }
          }
          ok = __all_sync(0xffffffffu, ok);
          from = to;
        }
        if (!ok) abort_flag = 1;
      }
    } else {
      // ---------------------------------------------------------- softmax
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
      const int t = warp >> 2;
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
      const uint32_t st = tmem + lanes + kTmemS + t * kTile, ot = tmem + lanes + kTmemO + t * HD;
      const int tiles = t ? job.tiles[1] : job.tiles[0], head = t ? job.head[1] : job.head[0];
      const int row = (t ? job.row0[1] : job.row0[0]) + (threadIdx.x & 127);
      const int seen = job.m - job.n + min(row, job.n - 1);  // the last key that the row sees
      const float c = a.scale_log2;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < tiles; ++j) {
        ok = __all_sync(0xffffffffu, wait(sbar + 8 * t, j & 1));
        if (!ok) break;
        fence_after();
        uint32_t v[kTile];
#pragma unroll
        for (int i = 0; i < kTile; i += 32) tmem_ld32(st + i, v + i);
        wait_ld();
        float* s = reinterpret_cast<float*>(v);
        const int lim = seen - j * kTile;
        if (__any_sync(0xffffffffu, lim < kTile - 1)) {
#pragma unroll
          for (int i = 0; i < kTile; ++i)
            if (i > lim) s[i] = -INFINITY;
        }
        float mx4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < kTile; i += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            mx4[e] = i + e + 4 < kTile ? fmaxf(fmaxf(mx4[e], s[i + e]), s[i + e + 4]) : fmaxf(mx4[e], s[i + e]);
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        mx = fmaxf(mx, m);
        const bool move = (mx - m) * c > kSlack;  // (also from -inf; false for NaN)
        if (__any_sync(0xffffffffu, move) && j > 0) {
          ok = __all_sync(0xffffffffu, wait(obar + 8 * t, (j - 1) & 1));
          if (!ok) break;
          fence_after();
          const float f = !move ? 1.f : m == -INFINITY ? 0.f : ex2((m - mx) * c);
          l *= f;
#pragma unroll
          for (int i = 0; i < HD; i += 32) {
            uint32_t o[32];
            tmem_ld32(ot + i, o);
            wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(ot + i, o);
          }
        }
        if (move) m = mx;
        const float mc = (m == -INFINITY ? 0.f : m * c) + kLower<T>;
        const uint64_t c2 = f2(c, c), mc2 = f2(-mc, -mc);
        uint64_t sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t p[kTile / 4];
#pragma unroll
          for (int i = 0; i < kTile / 4; ++i) {
            const int e = h * (kTile / 2) + 2 * i;
            const uint64_t x2 = fma2(f2(s[e], s[e + 1]), c2, mc2);
            float x, y;
            if ((i & 7) < kPoly) {
              ex2_poly<T>(x2, x, y);
            } else {
              f2_split(x2, x, y);
              x = ex2(x);
              y = ex2(y);
            }
            sum[i & 1] = add2(sum[i & 1], f2(x, y));
            p[i] = pack2<T>(x, y);
          }
          tmem_st32(st + 32 * h, p);
          wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0)
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pbar + 16 * t + 8 * h) : "memory");
        }
        float x, y;
        f2_split(add2(sum[0], sum[1]), x, y);
        l += x + y;
        if (!(x + y <= 3.4e38f)) l = __int_as_float(0x7fffffff);  // a NaN that the polynomial made a number of
      }
      if (ok && tiles > 0) ok = __all_sync(0xffffffffu, wait(obar + 8 * t, (tiles - 1) & 1));
      if (!ok) {
        abort_flag = 1;
        if (lane == 0) {
          atomicExch(&g_prompt_status, (unsigned)PF_ERR_TIMEOUT);
          if (a.status) atomicExch(a.status, (unsigned)PF_ERR_TIMEOUT);
        }
      }
      fence_after();
      T* out = static_cast<T*>(a.out) + (long long)(job.q0 + row) * a.os + (long long)head * a.hd;
      const bool mine = head >= 0 && row < job.n;
      const bool none = ok && seen < 0;  // no key seen: zeros (and 0 / 0 where every score is -inf)
      const float inv = ok ? 1.f / l : __int_as_float(0x7fffffff);
#pragma unroll
      for (int i = 0; i < HD; i += 32) {
        uint32_t o[32];
        __syncwarp();  // lanes may come from without_hidden
        if (ok && tiles > 0) {
          tmem_ld32(ot + i, o);
          wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (mine && i < a.hd) {
          float* const f = reinterpret_cast<float*>(o);
          float big = 0.f;
          bool nan = false;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if (none) f[e] = 0.f;
            big = fmaxf(big, fabsf(f[e]));
            nan = nan || f[e] != f[e];
          }
          // (a sum of weights that is not finite is the row's own: a score it sees is not)
          if ((nan || big > 3.4e38f) && ok && l <= 3.4e38f &&
              without_hidden<T>(a, job.q0 + row, head, job.k0, job.kvh, seen, min(job.m, tiles * kTile), i,
                                (m == -INFINITY ? 0.f : m * c) + kLower<T>, inv))
            continue;
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            if (i + e < a.hd) {
              uint4 w;
              const float g = none ? 1.f : inv;
              w.x = pack2<T>(f[e] * g, f[e + 1] * g);
              w.y = pack2<T>(f[e + 2] * g, f[e + 3] * g);
              w.z = pack2<T>(f[e + 4] * g, f[e + 5] * g);
              w.w = pack2<T>(f[e + 6] * g, f[e + 7] * g);
              *reinterpret_cast<uint4*>(out + i + e) = w;
            }
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (abort_flag) {  // block-uniform: raised before the barrier only
    const int never = 0;
    auto drain = [&](uint32_t bar, uint32_t parity) { bar_wait(bar, parity, &never, kPollMask, kWaitNs); };
    if (threadIdx.x == 32 * kTmaWarp && copies > 0) {  // (Q goes out in front of the first of them)
      drain(qbar, 0);
      for (int i = max(0, copies - kStages); i < copies; ++i) drain(full0 + 8 * (i % kStages), (i / kStages) & 1);
    }
    if (warp == kMmaWarp) {
      if (elect_one()) {  // the thread that issued the products: a commit covers its own
        commit(dbar);
        drain(dbar, 0);
      }
      __syncwarp();
    }
    fence_before();
    __syncthreads();
  }
  if (warp == kMmaWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// [rows][heads][hd] of 16-bit values, boxes of 64 columns of one head in kTile rows.
bool make_map(CUtensorMap* map, const void* p, bool bf16, int hd, int heads, int rows, long long stride) {
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)stride * 2};
  const cuuint32_t box[3] = {64, 1, kTile}, es[3] = {1, 1, 1};
  const auto fn = encode_fn();
  return fn && fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, typename T>
cudaError_t launch_prompt(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const PromptArgs& a,
                          unsigned blocks, cudaStream_t s) {
  constexpr auto kern = prompt_attn_kernel<HD, T>;
  const cudaError_t e = allow_smem<kern>(Cfg<HD>::kSmem);
  if (e != cudaSuccess) return e;
  return launch_pdl_smem(kern, dim3(blocks), kThreads, Cfg<HD>::kSmem, s, q, k, v, a);
}

}  // namespace
}  // namespace pfb

using namespace pfb;

static int prompt_attention(const void* q, long long q_stride, const void* k, long long k_stride, const void* v,
                            long long v_stride, void* out, long long out_stride, int dtype, const int* cu_q,
                            const int* cu_k, int seqs, int total_q, int total_k, int n_heads, int n_kv_heads,
                            int head_dim, float scale, int* status, unsigned poll_mask, unsigned long long wait_ns,
                            void* stream) {
  if (!q || !out || out == q || out == k || out == v || !cu_q || !cu_k || seqs < 0 || total_q < 0 || total_k < 0 || (total_k > 0 && (!k || !v)) ||
      !(scale > 0.f && scale <= 3e38f) || (dtype != PF_DTYPE_F16 && dtype != PF_DTYPE_BF16))
    return PF_ERR_INVALID_ARGUMENT;
  if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || n_heads > 65535 || head_dim <= 0 || head_dim > 128 ||
      head_dim % 8)
    return PF_ERR_SHAPE;
  const long long qr = (long long)n_heads * head_dim, kr = (long long)n_kv_heads * head_dim;
  if (q_stride < qr || out_stride < qr || k_stride < kr || v_stride < kr) return PF_ERR_SHAPE;
  // tensor maps: strides below 2^40 bytes
  if ((q_stride | k_stride | v_stride) >> 38 || out_stride >> 38) return PF_ERR_SHAPE;
  if (!al16(q) || !al16(k) || !al16(v) || !al16(out) || !al4(cu_q) || !al4(cu_k) || !al4(status) || q_stride % 8 ||
      k_stride % 8 || v_stride % 8 || out_stride % 8)
    return PF_ERR_ALIGNMENT;
  // no more pairs of tiles than this: every sequence but an empty one adds less than one tile per head to total_q / 128
  const long long G = n_heads / n_kv_heads, some = seqs < total_q ? seqs : total_q;
  const long long blocks = ((total_q / kTile + some) * G + some + 1) / 2 * n_kv_heads;
  if (blocks > 0x7fffffffLL) return PF_ERR_SHAPE;
  if (seqs == 0 || total_q == 0) return PF_OK;
  const bool bf16 = dtype == PF_DTYPE_BF16;
  CUtensorMap qm, km, vm;
  // without keys nothing is loaded: any valid map will do
  if (!make_map(&qm, q, bf16, head_dim, n_heads, total_q, q_stride) ||
      !make_map(&km, total_k ? k : q, bf16, head_dim, total_k ? n_kv_heads : n_heads, total_k ? total_k : total_q,
                total_k ? k_stride : q_stride) ||
      !make_map(&vm, total_k ? v : q, bf16, head_dim, total_k ? n_kv_heads : n_heads, total_k ? total_k : total_q,
                total_k ? v_stride : q_stride))
    return report_cuda(cudaErrorInvalidValue);
  const PromptArgs a{q, k, v, out, q_stride, k_stride, v_stride, out_stride, cu_q, cu_k, seqs, total_q, total_k, (int)G, n_kv_heads, head_dim,
                     scale * 1.4426950408889634f, reinterpret_cast<unsigned*>(status), poll_mask, wait_ns};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned n = (unsigned)blocks;
  const cudaError_t e =
      head_dim > 64 ? (bf16 ? launch_prompt<128, __nv_bfloat16>(qm, km, vm, a, n, s) : launch_prompt<128, __half>(qm, km, vm, a, n, s))
                    : (bf16 ? launch_prompt<64, __nv_bfloat16>(qm, km, vm, a, n, s) : launch_prompt<64, __half>(qm, km, vm, a, n, s));
  return e == cudaSuccess ? PF_OK : report_cuda(e);
}

int pf_prompt_attention(const void* q, long long q_stride, const void* k, long long k_stride, const void* v,
                        long long v_stride, void* out, long long out_stride, int dtype, const int* cu_q,
                        const int* cu_k, int seqs, int total_q, int total_k, int n_heads, int n_kv_heads,
                        int head_dim, float scale, int* status, void* stream) {
  return prompt_attention(q, q_stride, k, k_stride, v, v_stride, out, out_stride, dtype, cu_q, cu_k, seqs, total_q,
                          total_k, n_heads, n_kv_heads, head_dim, scale, status, kPollMask, kWaitNs, stream);
}

int pf_prompt_selftest(const void* q, long long q_stride, const void* k, long long k_stride, const void* v,
                       long long v_stride, void* out, long long out_stride, int dtype, const int* cu_q,
                       const int* cu_k, int seqs, int total_q, int total_k, int n_heads, int n_kv_heads, int head_dim,
                       float scale, int* status, unsigned long long wait_ns, void* stream) {
  if (wait_ns > kWaitNs) return PF_ERR_INVALID_ARGUMENT;
  return prompt_attention(q, q_stride, k, k_stride, v, v_stride, out, out_stride, dtype, cu_q, cu_k, seqs, total_q,
                          total_k, n_heads, n_kv_heads, head_dim, scale, status, 0, wait_ns, stream);
}

int pf_prompt_status(int reset, int* status, void* stream) {
  if (!status) return PF_ERR_INVALID_ARGUMENT;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  unsigned word = 0;
  cudaError_t e = cudaStreamSynchronize(s);
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(&word, g_prompt_status, sizeof(word), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e == cudaSuccess && reset && word) {
    const unsigned zero = 0;
    e = cudaMemcpyToSymbolAsync(g_prompt_status, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  }
  if (e != cudaSuccess) return report_cuda(e);
  *status = (int)word;
  return PF_OK;
}
