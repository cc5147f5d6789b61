// Attention of one new token per sequence over its cache.
//
// Reading the cache once bounds it.  A CTA owns one key head of one sequence
// (up to GC of the query heads that share it) and one slice of the keys; its
// warps take keys in turn, a lane holds 4 of the D columns, and every warp
// keeps its own running maximum, sum and output.  With few sequences the keys
// are split over CTAs whose partial results a second kernel joins in order.
#include "attention.cuh"

namespace kf {
namespace {

using namespace attn;

constexpr int kWarps = 4, kMaxSplits = 64;

struct DecodeArgs {
  const void* q;  // (B, H, D)
  const void* k;  // (B, capacity, KV, D), strides in elements
  const void* v;
  int64_t q_batch, q_head, k_batch, k_row, k_head, v_batch, v_row, v_head;
  const int* lengths;
  const void* table;
  const int* buckets;
  void* o;      // (B, H, D)
  float* part;  // (B, H, splits, D + 2): output, maximum, sum
  int batch, capacity, heads, kv_heads, dim, span, splits;
  bool table_bf16;
  float scale;
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(a.x << 16), v[1] = __uint_as_float(a.x & 0xffff0000u);
  v[2] = __uint_as_float(a.y << 16), v[3] = __uint_as_float(a.y & 0xffff0000u);
}

template <typename T, int GC>
__global__ void __launch_bounds__(kWarps * 32) attention_decode(const DecodeArgs a) {
  extern __shared__ float sbias[];  // GC x (2 span + 1)
  __shared__ float so[kWarps][GC][kMaxDim], sm[kWarps][GC], sl[kWarps][GC];
  const int group = a.heads / a.kv_heads, chunks = (group + GC - 1) / GC;
  const int split = blockIdx.x, kv_head = blockIdx.y / chunks, g0 = blockIdx.y % chunks * GC, b = blockIdx.z;
  const int n_g = min(GC, group - g0), head0 = kv_head * group + g0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = min(max(a.lengths[b], 0), a.capacity);
  const int per = ((len + a.splits - 1) / a.splits + 15) / 16 * 16;
  const int first = min(len, split * per), last = min(len, first + per);
  const int n_bias = 2 * a.span + 1;
  if (a.table != nullptr) {
    for (int i = threadIdx.x; i < n_g * n_bias; i += kWarps * 32) {
      const int64_t at = (int64_t)a.buckets[i % n_bias] * a.heads + head0 + i / n_bias;
      const float v = a.table_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.table)[at])
                                   : static_cast<const float*>(a.table)[at];
      sbias[i] = bias_base2(v);
    }
    __syncthreads();
  }
  const bool active = lane * 4 < a.dim;
  float q[GC][4], o[GC][4], m[GC], l[GC];
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    m[g] = -CUDART_INF_F, l[g] = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) q[g][c] = o[g][c] = 0.f;
    if (g < n_g && active) load4<T>(static_cast<const T*>(a.q) + b * a.q_batch + (head0 + g) * a.q_head + lane * 4, q[g]);
  }
  const T* kp = static_cast<const T*>(a.k) + b * a.k_batch + kv_head * a.k_head + lane * 4;
  const T* vp = static_cast<const T*>(a.v) + b * a.v_batch + kv_head * a.v_head + lane * 4;
  const float c2 = a.scale * kLog2e;
  constexpr int U = 4;  // keys in flight per warp
  for (int key0 = first + warp * U; key0 < last; key0 += kWarps * U) {
    float kk[U][4], vv[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int c = 0; c < 4; ++c) kk[u][c] = vv[u][c] = 0.f;
      if (active && key0 + u < last) {
        load4<T>(kp + (int64_t)(key0 + u) * a.k_row, kk[u]);
        load4<T>(vp + (int64_t)(key0 + u) * a.v_row, vv[u]);
      }
    }
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      float t[U], top = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        t[u] = q[g][0] * kk[u][0] + q[g][1] * kk[u][1] + q[g][2] * kk[u][2] + q[g][3] * kk[u][3];
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) t[u] += __shfl_xor_sync(0xffffffffu, t[u], s);
        t[u] *= c2;
        if (a.table != nullptr && g < n_g) t[u] += sbias[g * n_bias + clamp_dist(len - 1 - key0 - u, a.span)];
        if (key0 + u >= last) t[u] = -CUDART_INF_F;
        top = fmaxf(top, t[u]);
      }
      const float base = top == -CUDART_INF_F ? 0.f : top, fix = exp2f(m[g] - base);
      m[g] = top;
      l[g] *= fix;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[g][c] *= fix;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = exp2f(t[u] - base);
        l[g] += p;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[g][c] = fmaf(p, vv[u][c], o[g][c]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    if (lane == 0) sm[warp][g] = m[g], sl[warp][g] = l[g];
#pragma unroll
    for (int c = 0; c < 4; ++c) so[warp][g][lane * 4 + c] = o[g][c];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_g * a.dim; i += kWarps * 32) {
    const int g = i / a.dim, c = i % a.dim;
    float top = -CUDART_INF_F, sum = 0.f, out = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w][g]);
    const float base = top == -CUDART_INF_F ? 0.f : top;
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(sm[w][g] - base);
      sum = fmaf(sl[w][g], f, sum);
      out = fmaf(so[w][g][c], f, out);
    }
    const int64_t row = (int64_t)b * a.heads + head0 + g;
    if (a.splits == 1) {
      static_cast<T*>(a.o)[row * a.dim + c] = from_f32<T>(sum == 0.f ? 0.f : out / sum);
    } else {
      float* p = a.part + (row * a.splits + split) * (a.dim + 2);
      p[c] = out;
      if (c == 0) p[a.dim] = top, p[a.dim + 1] = sum;
    }
  }
}

// Joins the splits of one (sequence, head) per warp, in order.
template <typename T>
__global__ void __launch_bounds__(128) attention_decode_join(const DecodeArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (int64_t)a.batch * a.heads) return;
  const int lane = threadIdx.x & 31;
  const float* p = a.part + row * a.splits * (a.dim + 2);
  float top = -CUDART_INF_F;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, p[s * (a.dim + 2) + a.dim]);
  const float base = top == -CUDART_INF_F ? 0.f : top;
  float sum = 0.f, out[4] = {};
  for (int s = 0; s < a.splits; ++s) {
    const float f = exp2f(p[s * (a.dim + 2) + a.dim] - base);
    sum = fmaf(p[s * (a.dim + 2) + a.dim + 1], f, sum);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane + 32 * c < a.dim) out[c] = fmaf(p[s * (a.dim + 2) + lane + 32 * c], f, out[c]);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 32 * c < a.dim) static_cast<T*>(a.o)[row * a.dim + lane + 32 * c] = from_f32<T>(sum == 0.f ? 0.f : out[c] / sum);
}

constexpr int kGC = 4;

int split_count(int batch, int capacity, int heads, int kv_heads) {
  const int64_t ctas = (int64_t)batch * kv_heads * cdiv(heads / kv_heads, kGC);
  const int64_t want = cdiv(148 * 4, std::max<int64_t>(1, ctas));
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, cdiv(capacity, 64), kMaxSplits}));
}

template <typename T>
int launch(const DecodeArgs& a, cudaStream_t st) {
  const dim3 grid(a.splits, a.kv_heads * (unsigned)cdiv(a.heads / a.kv_heads, kGC), a.batch);
  const size_t smem = a.table != nullptr ? kGC * (2 * a.span + 1) * sizeof(float) : 0;
  auto* kernel = attention_decode<T, kGC>;
  KF_CUDA_RET(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<grid, kWarps * 32, smem, st>>>(a);
  if (int rc = check_launch("kf_attention_decode")) return rc;
  if (a.splits == 1) return KF_OK;
  attention_decode_join<T><<<(unsigned)cdiv((int64_t)a.batch * a.heads, 4), 128, 0, st>>>(a);
  return check_launch("kf_attention_decode");
}

}  // namespace
}  // namespace kf

extern "C" int kf_attention_decode_splits(const kf_decode_desc* d) {
  if (d == nullptr || d->kv_heads < 1 || d->batch < 1) return 1;
  return kf::split_count(d->batch, d->capacity, d->heads, d->kv_heads);
}

extern "C" int kf_attention_decode(const void* q, const void* k, const void* v, const int32_t* lengths, const void* table,
                                   const int32_t* buckets, void* o, float* workspace, const kf_decode_desc* d, void* stream) {
  using namespace kf;
  clear_error();
  const char* fn = "kf_attention_decode";
  KF_CHECK_ARG(d != nullptr, "%s: null descriptor", fn);
  KF_CHECK_ARG(d->heads >= 1 && d->kv_heads >= 1 && d->heads % d->kv_heads == 0, "%s: %d heads do not divide over %d key heads", fn,
               d->heads, d->kv_heads);
  KF_CHECK_ARG(d->dim >= 8 && d->dim <= attn::kMaxDim && d->dim % 8 == 0, "%s: head width %d is not a multiple of 8 up to %d", fn,
               d->dim, attn::kMaxDim);
  KF_CHECK_ARG(d->dtype == KF_DTYPE_F32 || d->dtype == KF_DTYPE_BF16, "%s: types must be float32 or bfloat16", fn);
  KF_CHECK_ARG(d->batch >= 0 && d->batch <= 65535 && d->capacity >= 0, "%s: bad sizes", fn);
  KF_CHECK_ARG(d->span >= 0 && d->span <= attn::kMaxSpan, "%s: bias distances up to %d are outside [0, %d]", fn, d->span, attn::kMaxSpan);
  if (d->batch == 0) return KF_OK;
  KF_CHECK_ARG(q && o && lengths && (d->capacity == 0 || (k && v)), "%s: null argument", fn);
  KF_CHECK_ARG((table == nullptr) == (buckets == nullptr), "%s: the bias needs a table and buckets", fn);
  if (int rc = bind_device(q)) return rc;
  DecodeArgs a{};
  a.q = q, a.k = k, a.v = v, a.lengths = lengths, a.table = table, a.buckets = buckets, a.o = o, a.part = workspace;
  a.q_batch = d->q_batch, a.q_head = d->q_head, a.k_batch = d->k_batch, a.k_row = d->k_row, a.k_head = d->k_head;
  a.v_batch = d->v_batch, a.v_row = d->v_row, a.v_head = d->v_head;
  a.batch = d->batch, a.capacity = d->capacity, a.heads = d->heads, a.kv_heads = d->kv_heads, a.dim = d->dim, a.span = d->span;
  a.splits = split_count(d->batch, d->capacity, d->heads, d->kv_heads);
  a.table_bf16 = d->table_dtype == KF_DTYPE_BF16, a.scale = d->scale;
  KF_CHECK_ARG(a.splits == 1 || workspace != nullptr, "%s: null workspace", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return d->dtype == KF_DTYPE_BF16 ? launch<__nv_bfloat16>(a, st) : launch<float>(a, st);
}
