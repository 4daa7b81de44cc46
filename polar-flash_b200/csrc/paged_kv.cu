// Paged KV cache: RoPE with the cache write for a batch of new tokens
// (pf_paged_rope_kv).  One warp handles one row of head_dim values (a query
// head, or a KV head's key or value) of one token:
//   (x[i], x[i + hd/2]) -> (x1 c - x2 s, x1 s + x2 c),
// every product and sum rounded on its own as pf_rope_kv rounds them, then
// the row is stored (16 or 32 bits) and, for keys and values, written into
// its page, quantized by the formulas of pf_kv_quantize.  Large calls are bound
// by memory where rows are 16 bits wide, by instructions where they are
// quantized (see launch_rope); small ones by a chain of four dependent reads
// (cu_seqlens, the lengths, the table, the row: 2.8 us for 64 tokens).
#include <math.h>

#include "common.cuh"
#include "launch.cuh"
#include "paged.cuh"

namespace pfb {
namespace {

constexpr int kRopeThreads = 256;
constexpr long long kManyRows = 16384;

struct RopeArgs {
  KvPages pages;
  const void *q, *k, *v;
  long long qs, ks, vs;  // elements between tokens
  const float *cos, *sin;
  const int *cu, *lens, *table;
  int tokens, width, seqs, nh;
  void *q_out, *k_out, *v_out;
};

template <int V>
struct Vec {
  float x[V];
};

// V consecutive values (V = 4 for head_dim 128, 2 for 64) from element `i`.
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[V]) {
  if constexpr (sizeof(T) == 4) {
    const Vec<V> v = *reinterpret_cast<const Vec<V>*>(__builtin_assume_aligned(p, 4 * V));
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = v.x[i];
  } else {
    T h[V];
    if constexpr (V == 4)
      *reinterpret_cast<uint2*>(h) = *reinterpret_cast<const uint2*>(p);
    else
      *reinterpret_cast<uint32_t*>(h) = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = to_f32(h[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[V]) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (V == 4)
      *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else
      *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
  } else {
    T h[V];
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = from_f32<T>(x[i]);
    if constexpr (V == 4)
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(h);
    else
      *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<uint32_t*>(h);
  }
}

// The warp's sequence of token t: the number of entries cu[1..seqs] that are
// <= t (cu ascending), found 32 entries at a time from both ends of a range
// that shrinks 33-fold per step.  Every read stays inside cu[0..seqs], whatever
// cu holds; the result is in 0..seqs (seqs: the token is behind the last one).
__device__ __forceinline__ int seq_of(const int* __restrict__ cu, int seqs, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = seqs;  // the answer is in lo..hi
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;  // probes at lo + step * (lane + 1), the last at most hi
    const int at = lo + step * (lane + 1);
    const bool below = at <= hi && cu[at] <= t;  // the answer is at least `at`
    const int n = __popc(__ballot_sync(0xffffffffu, below));
    const int nlo = lo + step * n;
    hi = min(hi, nlo + step - 1);
    lo = nlo;
  }
  return min(lo, seqs);
}

// Maxima and minima that hand NaN on, as the tensor expression's do: a row with a
// NaN has a NaN scale, and reads back as NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <int HD, int MODE>
__device__ __forceinline__ void write_row(const KvPages& pg, bool key, size_t row, const float (&x)[HD / 32]) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x & 31;
  uint8_t* base = static_cast<uint8_t*>(key ? pg.k : pg.v);
  if constexpr (MODE == PF_KV_F16) {
    store_vec(reinterpret_cast<__half*>(base) + row * HD + lane * V, x);
  } else if constexpr (MODE == PF_KV_BF16) {
    store_vec(reinterpret_cast<__nv_bfloat16*>(base) + row * HD + lane * V, x);
  } else {
    float lo = INFINITY, hi = MODE == PF_KV_2BIT_ASYM ? -INFINITY : 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      hi = max_nan(hi, MODE == PF_KV_2BIT_ASYM ? x[i] : fabsf(x[i]));
      lo = min_nan(lo, x[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      if (MODE == PF_KV_2BIT_ASYM) lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    // times the fp32 reciprocal, as torch divides by a number on a CUDA device (pf_kv_quantize
    // takes the quotient: its scale may be one rounding away)
    const float s = MODE == PF_KV_INT8   ? max_nan(__fmul_rn(hi, 1.f / 127.f), 1e-8f)
                    : MODE == PF_KV_2BIT ? max_nan(__fmul_rn(hi, 1.f / 1.75f), 1e-8f)
                                         : max_nan(__fmul_rn(__fsub_rn(hi, lo), 1.f / 3.f), 1e-8f);
    unsigned code = 0;  // the lane's V codes, packed as the row stores them
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (MODE == PF_KV_INT8) {
        const float r = fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -128.f), 127.f);
        code |= ((unsigned)(int)r & 0xffu) << (8 * i);
      } else {
        const float r =
            MODE == PF_KV_2BIT ? floorf(__fadd_rn(__fdiv_rn(x[i], s), 2.f)) : rintf(__fdiv_rn(__fsub_rn(x[i], lo), s));
        code |= (unsigned)fminf(fmaxf(r, 0.f), 3.f) << (2 * (V - 1 - i));
      }
    }
    uint8_t* dst = base + row * (MODE == PF_KV_INT8 ? HD : HD / 4);
    if constexpr (MODE == PF_KV_INT8) {
      if constexpr (V == 4)
        *reinterpret_cast<uint32_t*>(dst + 4 * lane) = code;
      else
        *reinterpret_cast<uint16_t*>(dst + 2 * lane) = (uint16_t)code;
    } else if constexpr (V == 4) {
      dst[lane] = (uint8_t)code;
    } else {  // two lanes share a byte, the even one's values in its top half
      const unsigned other = __shfl_xor_sync(0xffffffffu, code, 1);
      if (!(lane & 1)) dst[lane >> 1] = (uint8_t)(code << 4 | other);
    }
    if (lane == 0) {
      (key ? pg.k_scales : pg.v_scales)[row] = s;
      if (MODE == PF_KV_2BIT_ASYM) (key ? pg.k_zeros : pg.v_zeros)[row] = lo;
    }
  }
}

// R rows of one token per warp, all asked for before the first is used.
template <int HD, int MODE, typename TI, typename TO, int R>
__global__ void __launch_bounds__(kRopeThreads) paged_rope_kv_kernel(const RopeArgs a) {
  constexpr int V = HD / 32, HALF = HD / 2;
  pdl_enter();
  const int lane = threadIdx.x & 31, nkv = a.pages.nkv, rows = a.nh + 2 * nkv, per = (rows + R - 1) / R;
  const long long w = (long long)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
  const int t = (int)(w / per), r0 = (int)(w - (long long)t * per) * R;  // rows: query heads, then keys, then values
  if (t >= a.tokens) return;
  float x[R][V], c[V], s[V];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + i;
    if (r >= rows) break;
    const TI* src = r < a.nh         ? static_cast<const TI*>(a.q) + t * a.qs + (size_t)r * HD
                    : r < a.nh + nkv ? static_cast<const TI*>(a.k) + t * a.ks + (size_t)(r - a.nh) * HD
                                     : static_cast<const TI*>(a.v) + t * a.vs + (size_t)(r - a.nh - nkv) * HD;
    load_vec(src + lane * V, x[i]);
  }
  const bool turn = a.cos && r0 < a.nh + nkv;
  if (turn) {
    const size_t at = (size_t)t * HALF + (lane & 15) * V;
    load_vec(a.cos + at, c);
    load_vec(a.sin + at, s);
  }
  const int b = a.cu ? seq_of(a.cu, a.seqs, t) : t;
  if (b >= a.seqs) return;  // behind the last sequence
  long long pos = 0;
  if (r0 + R > a.nh) pos = (long long)a.lens[b] - ((long long)(a.cu ? a.cu[b + 1] : t + 1) - t);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + i;
    if (r >= rows) break;
    const bool is_q = r < a.nh, is_k = !is_q && r < a.nh + nkv;
    const int head = is_q ? r : is_k ? r - a.nh : r - a.nh - nkv;
    if (turn && (is_q || is_k)) {
      // lanes 0..15 hold the first half of the row, lanes 16..31 the second
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float y = __shfl_xor_sync(0xffffffffu, x[i][e], 16);
        x[i][e] = lane < 16 ? __fsub_rn(__fmul_rn(x[i][e], c[e]), __fmul_rn(y, s[e]))
                            : __fadd_rn(__fmul_rn(y, s[e]), __fmul_rn(x[i][e], c[e]));
      }
    }
    void* out = is_q ? a.q_out : is_k ? a.k_out : a.v_out;
    if (out) store_vec(static_cast<TO*>(out) + ((size_t)t * (is_q ? a.nh : nkv) + head) * HD + lane * V, x[i]);
    if (is_q) continue;
    const long long row = page_row(a.pages, a.table, a.width, b, head, pos);
    if (row >= 0) write_row<HD, MODE>(a.pages, is_k, (size_t)row, x[i]);
  }
}

// Four rows per warp where the rows fill the machine more than once, one where
// the call is short of warps.  48 rows of 128 per token into int8 pages, one
// and four rows per warp: 64 tokens 3.7 and 5.0 us, 256 5.8 and 6.1, 700 11.5
// and 10.2, 8000 99.5 and 73.7.  Of that call the bytes are 49 us at the copy rate,
// and the same into bf16 pages, 332 MB for 316, takes 62 us: what bounds it is
// its instructions, 168 a row, 0.79 issued a cycle and scheduler.
template <int HD, int MODE, typename TI, typename TO>
cudaError_t launch_rope(const RopeArgs& a, cudaStream_t s) {
  const long long rows = a.nh + 2 * a.pages.nkv, warps = kRopeThreads / 32;
  if (a.tokens * rows >= kManyRows) {
    const long long n = a.tokens * ((rows + 3) / 4);
    return launch_pdl(paged_rope_kv_kernel<HD, MODE, TI, TO, 4>, dim3((unsigned)((n + warps - 1) / warps)), kRopeThreads, s, a);
  }
  const long long n = a.tokens * rows;
  return launch_pdl(paged_rope_kv_kernel<HD, MODE, TI, TO, 1>, dim3((unsigned)((n + warps - 1) / warps)), kRopeThreads, s, a);
}

template <int HD, int MODE, typename TI>
cudaError_t launch_rope(const RopeArgs& a, int out_dtype, cudaStream_t s) {
  if (out_dtype == PF_DTYPE_F16) return launch_rope<HD, MODE, TI, __half>(a, s);
  if (out_dtype == PF_DTYPE_BF16) return launch_rope<HD, MODE, TI, __nv_bfloat16>(a, s);
  return launch_rope<HD, MODE, TI, float>(a, s);
}

template <int HD, int MODE>
cudaError_t launch_rope(const RopeArgs& a, int dtype, int out_dtype, cudaStream_t s) {
  if (dtype == PF_DTYPE_F16) return launch_rope<HD, MODE, __half>(a, out_dtype, s);
  if (dtype == PF_DTYPE_BF16) return launch_rope<HD, MODE, __nv_bfloat16>(a, out_dtype, s);
  return launch_rope<HD, MODE, float>(a, out_dtype, s);
}

template <int HD>
cudaError_t launch_rope(const RopeArgs& a, int mode, int dtype, int out_dtype, cudaStream_t s) {
  switch (mode) {
    case PF_KV_INT8: return launch_rope<HD, PF_KV_INT8>(a, dtype, out_dtype, s);
    case PF_KV_2BIT: return launch_rope<HD, PF_KV_2BIT>(a, dtype, out_dtype, s);
    case PF_KV_2BIT_ASYM: return launch_rope<HD, PF_KV_2BIT_ASYM>(a, dtype, out_dtype, s);
    case PF_KV_F16: return launch_rope<HD, PF_KV_F16>(a, dtype, out_dtype, s);
    default: return launch_rope<HD, PF_KV_BF16>(a, dtype, out_dtype, s);
  }
}

bool dtype_ok(int d) { return d == PF_DTYPE_F32 || d == PF_DTYPE_F16 || d == PF_DTYPE_BF16; }

}  // namespace
}  // namespace pfb

using namespace pfb;

int pf_kv_pages_check(const pf_kv_pages* p) {
  if (!p || !p->k || !p->v) return PF_ERR_INVALID_ARGUMENT;
  const bool coded = p->mode == PF_KV_INT8 || p->mode == PF_KV_2BIT || p->mode == PF_KV_2BIT_ASYM;
  if (!coded && p->mode != PF_KV_F16 && p->mode != PF_KV_BF16) return PF_ERR_INVALID_ARGUMENT;
  if (coded && (!p->k_scales || !p->v_scales)) return PF_ERR_INVALID_ARGUMENT;
  if (p->mode == PF_KV_2BIT_ASYM && (!p->k_zeros || !p->v_zeros)) return PF_ERR_INVALID_ARGUMENT;
  if (p->num_pages <= 0 || p->n_kv_heads <= 0 || p->n_kv_heads > 65535) return PF_ERR_SHAPE;
  if (p->head_dim != 64 && p->head_dim != 128) return PF_ERR_SHAPE;
  const int ps = p->page_size;
  if (ps != 16 && ps != 32 && ps != 64 && ps != 128 && ps != 256) return PF_ERR_SHAPE;
  if (!al16(p->k) || !al16(p->v)) return PF_ERR_ALIGNMENT;
  if (coded && (!al16(p->k_scales) || !al16(p->v_scales))) return PF_ERR_ALIGNMENT;
  if (p->mode == PF_KV_2BIT_ASYM && (!al16(p->k_zeros) || !al16(p->v_zeros))) return PF_ERR_ALIGNMENT;
  return PF_OK;
}

int pf_paged_rope_kv(const pf_kv_pages* pages, const void* q, long long q_stride, const void* k, long long k_stride,
                     const void* v, long long v_stride, int dtype, const float* cos, const float* sin, int tokens,
                     const int* cu_seqlens, const int* seq_lens, const int* block_table, int table_width, int seqs,
                     int n_heads, void* q_out, void* k_out, void* v_out, int out_dtype, void* stream) {
  const int st = pf_kv_pages_check(pages);
  if (st != PF_OK) return st;
  if (!dtype_ok(dtype) || !dtype_ok(out_dtype) || tokens < 0 || seqs < 0) return PF_ERR_INVALID_ARGUMENT;
  if (!k || !v || !seq_lens || !block_table || !cos != !sin || n_heads < 0 || (n_heads > 0) != (q != nullptr) ||
      (n_heads > 0) != (q_out != nullptr) || !k_out != !v_out)
    return PF_ERR_INVALID_ARGUMENT;
  const int nkv = pages->n_kv_heads, hd = pages->head_dim;
  if (n_heads > 65535 || table_width <= 0 || (!cu_seqlens && tokens != seqs)) return PF_ERR_SHAPE;
  // whole rows, and 16-byte steps from token to token
  const int per16 = dtype == PF_DTYPE_F32 ? 4 : 8;
  if ((n_heads && q_stride < (long long)n_heads * hd) || k_stride < (long long)nkv * hd ||
      v_stride < (long long)nkv * hd)
    return PF_ERR_SHAPE;
  if ((n_heads && q_stride % per16) || k_stride % per16 || v_stride % per16) return PF_ERR_ALIGNMENT;
  if (!al16(q) || !al16(k) || !al16(v) || !al16(cos) || !al16(sin) || !al16(q_out) || !al16(k_out) || !al16(v_out) ||
      !al4(cu_seqlens) || !al4(seq_lens) || !al4(block_table))
    return PF_ERR_ALIGNMENT;
  if (q && q == q_out && (dtype != out_dtype || q_stride != (long long)n_heads * hd)) return PF_ERR_INVALID_ARGUMENT;
  if (tokens == 0 || seqs == 0) return PF_OK;
  if ((long long)tokens * (n_heads + 2 * nkv) > 0x7fffffffLL) return PF_ERR_SHAPE;
  RopeArgs a{};
  a.pages = kv_pages(*pages);
  a.q = q;
  a.k = k;
  a.v = v;
  a.qs = q_stride;
  a.ks = k_stride;
  a.vs = v_stride;
  a.cos = cos;
  a.sin = sin;
  a.cu = cu_seqlens;
  a.lens = seq_lens;
  a.table = block_table;
  a.tokens = tokens;
  a.width = table_width;
  a.seqs = seqs;
  a.nh = n_heads;
  a.q_out = q_out;
  a.k_out = k_out;
  a.v_out = v_out;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = hd == 128 ? launch_rope<128>(a, pages->mode, dtype, out_dtype, s)
                                  : launch_rope<64>(a, pages->mode, dtype, out_dtype, s);
  return e == cudaSuccess ? PF_OK : report_cuda(e);
}
