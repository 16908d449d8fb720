// Per-head RMS norms of q and k, RoPE of both and the K/V append in one pass (include/pkv.h,
// "QK norm + RoPE + append").
//
// A head x of D values becomes  y[i] = x[i] / sqrt(mean(x^2) + eps) * w[i], then the rotation of
// rope_append.cu: y'[i] = y[i] c[i] - y[i + D/2] s[i], y'[i + D/2] = y[i + D/2] c[i] + y[i] s[i].  All of it in
// fp32, rounded to the element type once, on the way out.
//
// The rows are read once and written once, so a large step is bound by HBM and a small one by the launch.
// D / 2 / (16 bytes) neighbouring lanes hold a head, each a 16-byte piece of either half: a lane owns whole
// rotation pairs, the sum of squares is a few shuffles inside the lanes of the head, and every load and store is
// 16 bytes.  A v head is a head without the arithmetic.  Steps that fill the GPU give a lane the same piece of two heads of
// one token, which share the token's cos / sin: 8,191 tokens of 32/8 heads of 128, bf16 (206 MB), 48 us with one head a
// lane, 43 with two, 71 with four (94 registers).  Steps whose rows do not fit L2 read and write them as data that is
// not used again: 36.5 us, 5.6 TB/s.  (The same rows again and again, kept and streamed: 2,048 tokens, 50 MB, 9.6 us both; 4,096,
// 101 MB, 21.4 and 18.2.  Below the border the launch behind finds its q, K and V in L2.)  Sending for the rows before the position is known: 36.2 -> 38.2 us.
#include "common.cuh"
#include "launch_util.hpp"
#include "status.hpp"

namespace pkv {
namespace {

constexpr int kNormThreads = 128;

template <typename T>
struct NormArgs {
  const T *q, *k, *v;
  long long q_stride, k_stride, v_stride;      // elements from one token's row to the next
  const T *q_weight, *k_weight;
  float eps;
  const int* positions;
  const float *cos_table, *sin_table;
  int max_positions;
  const int* slots;
  long long n_slots;
  T *q_out, *k_cache, *v_cache;
  int n_tokens, q_heads, kv_heads, head_dim;
};

// Head `head` of a token among its q, k and v heads: where it is read from, and where it goes (null: nowhere).
template <typename T>
__device__ __forceinline__ void head_rows(const NormArgs<T>& a, int token, int head, int slot, const T*& src, T*& dst) {
  const int hd = a.head_dim;
  const bool stored = slot >= 0 && slot < a.n_slots;
  if (head < a.q_heads) {
    src = a.q + token * a.q_stride + static_cast<long long>(head) * hd;
    dst = a.q_out + (static_cast<long long>(token) * a.q_heads + head) * hd;
  } else if (head < a.q_heads + a.kv_heads) {
    const int h = head - a.q_heads;
    src = a.k + token * a.k_stride + static_cast<long long>(h) * hd;
    dst = stored ? a.k_cache + (static_cast<long long>(slot) * a.kv_heads + h) * hd : nullptr;
  } else {
    const int h = head - a.q_heads - a.kv_heads;
    src = a.v + token * a.v_stride + static_cast<long long>(h) * hd;
    dst = stored ? a.v_cache + (static_cast<long long>(slot) * a.kv_heads + h) * hd : nullptr;
  }
}

template <typename T>
__device__ __forceinline__ void widen(const uint4& x, float (&f)[16 / sizeof(T)]) {
  const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) f[i] = Elem<T>::to_f32(e[i]);
}

template <typename T>
__device__ __forceinline__ void load_floats(const float* p, float (&f)[16 / sizeof(T)]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); i += 4) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(p + i));
    f[i] = x.x; f[i + 1] = x.y; f[i + 2] = x.z; f[i + 3] = x.w;
  }
}

// LANES lanes a head, HEADS heads a lane; STREAM: nothing is kept in L2.  q_out may be q: a lane reads the pieces it writes before it writes them.
template <typename T, int LANES, int HEADS, bool STREAM>
__global__ void __launch_bounds__(kNormThreads) qk_norm_rope_kernel(const NormArgs<T> a) {
  constexpr int E = 16 / sizeof(T);
  pdl_launch_dependents();
  pdl_wait();
  const unsigned heads = a.q_heads + 2 * a.kv_heads, per_token = (heads + HEADS - 1) / HEADS;
  const unsigned group = blockIdx.x * (kNormThreads / LANES) + threadIdx.x / LANES, at = group / per_token;
  // lanes of a group leave together, and so do whole warps of them or not: the shuffles below name the group's lanes
  if (at >= static_cast<unsigned>(a.n_tokens)) return;
  const int token = static_cast<int>(at), head0 = static_cast<int>(group - at * per_token) * HEADS;
  const int piece = threadIdx.x % LANES, half = a.head_dim / 2;
  const unsigned lanes = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1u) << ((threadIdx.x & 31) / LANES * LANES);
  const int pos = __ldg(a.positions + token), slot = a.kv_heads > 0 ? __ldg(a.slots + token) : -1;
  if (pos < 0 || pos >= a.max_positions) return;                 // a padding row: untouched

  uint4 lo[HEADS], hi[HEADS];
  T* dst[HEADS];
#pragma unroll
  for (int u = 0; u < HEADS; ++u) {
    dst[u] = nullptr;
    lo[u] = hi[u] = make_uint4(0u, 0u, 0u, 0u);
    if (head0 + u < static_cast<int>(heads)) {
      const T* src;
      head_rows(a, token, head0 + u, slot, src, dst[u]);
      // plain loads: q_out may be q
      const uint4 *x = reinterpret_cast<const uint4*>(src + piece * E), *y = reinterpret_cast<const uint4*>(src + half + piece * E);
      lo[u] = STREAM ? __ldcs(x) : *x;
      hi[u] = STREAM ? __ldcs(y) : *y;
    }
  }
  float c[E], s[E];
  const long long t = static_cast<long long>(pos) * half + piece * E;
  load_floats<T>(a.cos_table + t, c);
  load_floats<T>(a.sin_table + t, s);
#pragma unroll
  for (int u = 0; u < HEADS; ++u) {
    const int head = head0 + u;
    if (head < a.q_heads + a.kv_heads) {
      float x[E], y[E], wx[E], wy[E], sum = 0.f;
      widen<T>(lo[u], x);
      widen<T>(hi[u], y);
#pragma unroll
      for (int i = 0; i < E; ++i) sum = fmaf(x[i], x[i], fmaf(y[i], y[i], sum));
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(lanes, sum, o);
      const float inv = __frsqrt_rn(sum / static_cast<float>(a.head_dim) + a.eps);
      const T* w = head < a.q_heads ? a.q_weight : a.k_weight;
      widen<T>(__ldg(reinterpret_cast<const uint4*>(w + piece * E)), wx);
      widen<T>(__ldg(reinterpret_cast<const uint4*>(w + half + piece * E)), wy);
      T* ox = reinterpret_cast<T*>(&lo[u]);
      T* oy = reinterpret_cast<T*>(&hi[u]);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float n = x[i] * inv * wx[i], m = y[i] * inv * wy[i];
        ox[i] = Elem<T>::from_f32(n * c[i] - m * s[i]);
        oy[i] = Elem<T>::from_f32(m * c[i] + n * s[i]);
      }
    }
    if (dst[u]) {
      uint4 *x = reinterpret_cast<uint4*>(dst[u] + piece * E), *y = reinterpret_cast<uint4*>(dst[u] + half + piece * E);
      if (STREAM) {
        __stcs(x, lo[u]);
        __stcs(y, hi[u]);
      } else {
        *x = lo[u];
        *y = hi[u];
      }
    }
  }
}

// Any even head_dim, any alignment and strides: a warp a head, a rotation pair a lane at a time.  An element a load, rows read
// twice: 8,191 tokens of 32/8 heads of 96, bf16, 182 us (a copy of the rows 24), 256 tokens 5.8.
template <typename T>
__global__ void __launch_bounds__(kNormThreads) qk_norm_rope_pairs_kernel(const NormArgs<T> a) {
  pdl_launch_dependents();
  pdl_wait();
  const int heads = a.q_heads + 2 * a.kv_heads, half = a.head_dim / 2, lane = threadIdx.x & 31;
  const long long total = static_cast<long long>(a.n_tokens) * heads;
  for (long long w = (blockIdx.x * static_cast<long long>(kNormThreads) + threadIdx.x) / 32; w < total;
       w += static_cast<long long>(gridDim.x) * (kNormThreads / 32)) {
    const int token = static_cast<int>(w / heads), head = static_cast<int>(w - static_cast<long long>(token) * heads);
    const int pos = a.positions[token], slot = a.kv_heads > 0 ? a.slots[token] : -1;
    if (pos < 0 || pos >= a.max_positions) continue;
    const T* src;
    T* dst;
    head_rows(a, token, head, slot, src, dst);
    if (head >= a.q_heads + a.kv_heads) {
      if (dst)
        for (int i = lane; i < a.head_dim; i += 32) dst[i] = src[i];
      continue;
    }
    float sum = 0.f;
    for (int i = lane; i < a.head_dim; i += 32) {
      const float x = Elem<T>::to_f32(src[i]);
      sum = fmaf(x, x, sum);
    }
    const float inv = __frsqrt_rn(warp_sum(sum) / static_cast<float>(a.head_dim) + a.eps);
    const T* weight = head < a.q_heads ? a.q_weight : a.k_weight;
    const float* cs = a.cos_table + static_cast<long long>(pos) * half;
    const float* sn = a.sin_table + static_cast<long long>(pos) * half;
    if (!dst) continue;
    for (int i = lane; i < half; i += 32) {
      const float x = Elem<T>::to_f32(src[i]) * inv * Elem<T>::to_f32(weight[i]);
      const float y = Elem<T>::to_f32(src[i + half]) * inv * Elem<T>::to_f32(weight[i + half]);
      dst[i] = Elem<T>::from_f32(x * cs[i] - y * sn[i]);
      dst[i + half] = Elem<T>::from_f32(y * cs[i] + x * sn[i]);
    }
  }
}

constexpr int kHeadsEach = 2;
constexpr long long kManyLanes = 148ll * 2048;              // more lanes than the GPU holds at once
constexpr long long kStreamBytes = 96ll << 20;              // of rows read and written

template <typename T, int LANES>
void launch_lanes(const NormArgs<T>& a, cudaStream_t stream) {
  const int heads = a.q_heads + 2 * a.kv_heads;
  auto blocks = [&](int each) {
    const long long groups = static_cast<long long>(a.n_tokens) * ((heads + each - 1) / each), per_block = kNormThreads / LANES;
    return dim3(static_cast<unsigned>((groups + per_block - 1) / per_block));
  };
  const long long all = static_cast<long long>(a.n_tokens) * heads;
  if (2 * all * a.head_dim * static_cast<long long>(sizeof(T)) > kStreamBytes)
    launch_pdl(qk_norm_rope_kernel<T, LANES, kHeadsEach, true>, blocks(kHeadsEach), dim3(kNormThreads), 0, stream, a);
  else if (all * LANES > kManyLanes)
    launch_pdl(qk_norm_rope_kernel<T, LANES, kHeadsEach, false>, blocks(kHeadsEach), dim3(kNormThreads), 0, stream, a);
  else
    launch_pdl(qk_norm_rope_kernel<T, LANES, 1, false>, blocks(1), dim3(kNormThreads), 0, stream, a);
}

template <typename T>
int qk_norm_rope_impl(const void* q, const void* k, const void* v, long long q_stride, long long k_stride, long long v_stride,
                      const void* q_weight, const void* k_weight, float eps, const int* positions, const float* cos_table,
                      const float* sin_table, int max_positions, const int* slots, void* q_out, void* k_cache, void* v_cache,
                      long long n_slots, int n_tokens, int q_heads, int kv_heads, int head_dim, pkv_stream stream) {
  const char* fn = "pkv_qk_norm_rope_append";
  if (n_tokens <= 0 || head_dim <= 0 || (q_heads <= 0 && kv_heads <= 0)) return PKV_OK;   // as pkv_rope_append
  if (q_heads < 0 || kv_heads < 0) return fail(PKV_E_ARG, "%s: negative head count", fn);
  if (head_dim % 2) return fail(PKV_E_UNSUPPORTED, "%s: head_dim %d must be even (rotation pairs)", fn, head_dim);
  if (!(eps >= 0.f)) return fail(PKV_E_ARG, "%s: eps must not be negative", fn);
  if (!positions || !cos_table || !sin_table || max_positions <= 0) return fail(PKV_E_ARG, "%s: null positions, or null or empty tables", fn);
  if (q_heads > 0 && (!q || !q_weight || !q_out)) return fail(PKV_E_ARG, "%s: null q, q_weight or q_out", fn);
  if (kv_heads > 0 && (!k || !v || !k_weight || !slots || !k_cache || !v_cache)) return fail(PKV_E_ARG, "%s: null K/V pointer", fn);
  const long long q_dim = static_cast<long long>(q_heads) * head_dim, kv_dim = static_cast<long long>(kv_heads) * head_dim;
  if (n_tokens > 1 && ((q_heads > 0 && q_stride < q_dim) || (kv_heads > 0 && (k_stride < kv_dim || v_stride < kv_dim))))
    return fail(PKV_E_ARG, "%s: row strides %lld, %lld, %lld are shorter than the rows (%lld, %lld, %lld)", fn, q_stride, k_stride,
                v_stride, q_dim, kv_dim, kv_dim);
  if (kv_heads > 0 && n_slots <= 0) return fail(PKV_E_ARG, "%s: n_slots %lld must be > 0", fn, n_slots);
  if (q_heads > 0 && q_out == q && n_tokens > 1 && q_stride != q_dim)
    return fail(PKV_E_ARG, "%s: q_out may be q only if q's rows are contiguous", fn);
  NormArgs<T> a;
  a.q = static_cast<const T*>(q); a.k = static_cast<const T*>(k); a.v = static_cast<const T*>(v);
  a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.q_weight = static_cast<const T*>(q_weight); a.k_weight = static_cast<const T*>(k_weight);
  a.eps = eps;
  a.positions = positions; a.cos_table = cos_table; a.sin_table = sin_table; a.max_positions = max_positions;
  a.slots = slots; a.n_slots = n_slots;
  a.q_out = static_cast<T*>(q_out); a.k_cache = static_cast<T*>(k_cache); a.v_cache = static_cast<T*>(v_cache);
  a.n_tokens = n_tokens; a.q_heads = q_heads; a.kv_heads = kv_heads; a.head_dim = head_dim;
  constexpr int E = 16 / sizeof(T);
  const int lanes = head_dim % (2 * E) == 0 ? head_dim / (2 * E) : 0;
  auto rows16 = [](const void* p, long long stride) { return aligned16(p) && (stride * static_cast<long long>(sizeof(T))) % 16 == 0; };
  const bool vec = aligned16(cos_table) && aligned16(sin_table) && aligned16(q_weight) && aligned16(k_weight) && aligned16(q_out) &&
                   aligned16(k_cache) && aligned16(v_cache) && (q_heads == 0 || rows16(q, n_tokens > 1 ? q_stride : 0)) &&
                   (kv_heads == 0 || (rows16(k, n_tokens > 1 ? k_stride : 0) && rows16(v, n_tokens > 1 ? v_stride : 0)));
  const long long heads = static_cast<long long>(q_heads) + 2ll * kv_heads;
  if (heads * n_tokens > 0x7fffffffll - kNormThreads)
    return fail(PKV_E_UNSUPPORTED, "%s: %d tokens of %lld heads; at most 2^31 heads a call", fn, n_tokens, heads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (vec && lanes == 4) launch_lanes<T, 4>(a, s);
  else if (vec && lanes == 8) launch_lanes<T, 8>(a, s);
  else if (vec && lanes == 16) launch_lanes<T, 16>(a, s);
  else if (vec && lanes == 32) launch_lanes<T, 32>(a, s);
  else {
    long long blocks = (static_cast<long long>(n_tokens) * heads + kNormThreads / 32 - 1) / (kNormThreads / 32);
    if (blocks > 148 * 16) blocks = 148 * 16;
    launch_pdl(qk_norm_rope_pairs_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(kNormThreads), 0, s, a);
  }
  return check_launch("qk_norm_rope_kernel");
}

}  // namespace
}  // namespace pkv

#define PKV_QK_NORM_ROPE(SUFFIX, TYPE)                                                                                            \
  int pkv_qk_norm_rope_append_##SUFFIX(const void* q, const void* k, const void* v, long long q_stride, long long k_stride,       \
                                       long long v_stride, const void* q_weight, const void* k_weight, float eps,                 \
                                       const int* positions, const float* cos_table, const float* sin_table, int max_positions,   \
                                       const int* slots, void* q_out, void* k_cache, void* v_cache, long long n_slots,            \
                                       int n_tokens, int q_heads, int kv_heads, int head_dim, pkv_stream stream) {                \
    return pkv::qk_norm_rope_impl<TYPE>(q, k, v, q_stride, k_stride, v_stride, q_weight, k_weight, eps, positions, cos_table,     \
                                        sin_table, max_positions, slots, q_out, k_cache, v_cache, n_slots, n_tokens, q_heads,     \
                                        kv_heads, head_dim, stream);                                                              \
  }
extern "C" {
PKV_QK_NORM_ROPE(f16, __half)
PKV_QK_NORM_ROPE(bf16, __nv_bfloat16)
PKV_QK_NORM_ROPE(f32, float)
}
