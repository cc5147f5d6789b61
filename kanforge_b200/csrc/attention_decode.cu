// Attention of one new token per sequence over its cache.
//
// Reading the cache once bounds it.  A CTA owns one key head of one sequence
// with up to 16 (bf16) or 4 (float32) of the query heads that share it, and one
// slice of the keys; the slices of a sequence are a thread block cluster, whose
// CTAs read each other's partial results from shared memory and write the output
// in one launch, in slice order.
//
// bf16 runs on mma.sync m16n8k16: the 16 rows are query heads, and one token
// would leave most rows of a 128-row tcgen05 tile empty.  The contraction over D
// and the columns of the output may be taken in any order, so lane (n, t) = (lane / 4, lane % 4) reads 16 bytes of K
// row n at 32 i + 8 t and 16 bytes of V rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9 at
// 64 h + 8 n: whole sectors.  Every lane copies what it will use itself into a
// ring in shared memory (cp.async, 16 keys to a stage), so that two stages are
// under way behind the one in use and no lane waits for another.  P enters as
// the sum of two bf16 numbers (16 bits of it): twice the products, which a kernel
// bound by memory has free, and no rounding of P.  48 caches of 1 to 8192 slots, 32
// heads of 128 on 8 key heads: 0.19 ms, 4.6 TB/s (0.70 of the measured copy rate;
// 0.24 ms with loads into registers); 700 slots of one sequence, 12 heads of 64: 7 us,
// most of it the launch, one trip to memory and the join.
//
// float32 runs on the CUDA cores: a lane holds 4 of the D columns, a warp takes
// 4 keys at a time (7 caches of up to 600 slots, 5 heads of 40: 12 us).
#include <cooperative_groups.h>

#include <climits>

#include "attention.cuh"

namespace kf {
namespace {

using namespace attn;
namespace cg = cooperative_groups;

constexpr int kWarps = 4, kMaxSplits = 16;

struct DecodeArgs {
  const void* q;  // (B, H, D)
  const void* k;  // (B, capacity, KV, D), strides in elements
  const void* v;
  int64_t q_batch, q_head, k_batch, k_row, k_head, v_batch, v_row, v_head;
  const int* lengths;
  const void* table;
  const int* buckets;
  void* o;  // (B, H, D)
  int capacity, heads, kv_heads, dim, span, n_buckets;
  bool table_bf16;
  float scale;
};

// What a CTA works on.
template <int GC>
struct Part {
  int b, kv_head, head0, n_g, len, first, last;

  __device__ explicit Part(const DecodeArgs& a) {
    const int group = a.heads / a.kv_heads, chunks = (group + GC - 1) / GC, splits = gridDim.x;
    const int chunk = blockIdx.y % chunks;
    b = blockIdx.z, kv_head = blockIdx.y / chunks;
    head0 = kv_head * group + chunk * GC, n_g = min(GC, group - chunk * GC);
    len = min(max(a.lengths[b], 0), a.capacity);
    const int per = ((len + splits - 1) / splits + 15) / 16 * 16;
    first = min(len, (int)blockIdx.x * per), last = min(len, first + per);
  }
};

// The biases that this CTA's keys need, in base 2: (n_g, 2 span + 1).
template <int GC>
__device__ __forceinline__ void load_bias(const DecodeArgs& a, const Part<GC>& p, float* sbias) {
  if (a.table == nullptr || p.first >= p.last) return;
  const int lo = clamp_dist(p.len - p.last, a.span), n = clamp_dist(p.len - 1 - p.first, a.span) - lo + 1;
  for (int i = threadIdx.x; i < n; i += kWarps * 32) {
    const int64_t at = (int64_t)min(max(a.buckets[lo + i], 0), a.n_buckets - 1) * a.heads + p.head0;
    for (int g = 0; g < p.n_g; ++g)
      sbias[g * (2 * a.span + 1) + lo + i] = bias_base2(a.table_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.table)[at + g])
                                                                     : static_cast<const float*>(a.table)[at + g]);
  }
}

// A warp's running state per head; the CTA's warps and then the cluster's CTAs
// join theirs.
template <int GC>
struct Partial {
  float o[kWarps][GC][kMaxDim];
  float m[kWarps][GC], l[kWarps][GC];
  float co[GC][kMaxDim], cm[GC], cl[GC];  // the CTA's
};

template <typename T, int GC>
__device__ __forceinline__ void join(const DecodeArgs& a, const Part<GC>& part, Partial<GC>* s) {
  __syncthreads();
  for (int i = threadIdx.x; i < part.n_g * a.dim; i += kWarps * 32) {
    const int g = i / a.dim, c = i - g * a.dim;
    float top = s->m[0][g], sum = 0.f, out = 0.f;
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s->m[w][g]);
    const float base = top == -CUDART_INF_F ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(s->m[w][g] - base);
      sum = fmaf(s->l[w][g], f, sum);
      out = fmaf(s->o[w][g][c], f, out);
    }
    if (gridDim.x == 1) {
      static_cast<T*>(a.o)[((int64_t)part.b * a.heads + part.head0 + g) * a.dim + c] = from_f32<T>(sum == 0.f ? 0.f : out / sum);
    } else {
      s->co[g][c] = out;
      if (c == 0) s->cm[g] = top, s->cl[g] = sum;
    }
  }
  if (gridDim.x == 1) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int splits = gridDim.x, rank = blockIdx.x;
  for (int i = rank * kWarps * 32 + threadIdx.x; i < part.n_g * a.dim; i += splits * kWarps * 32) {
    const int g = i / a.dim, c = i - g * a.dim;
    float top = -CUDART_INF_F, sum = 0.f, out = 0.f;
    for (int r = 0; r < splits; ++r) top = fmaxf(top, *cluster.map_shared_rank(&s->cm[g], r));
    const float base = top == -CUDART_INF_F ? 0.f : top;
    for (int r = 0; r < splits; ++r) {
      const float f = exp2f(*cluster.map_shared_rank(&s->cm[g], r) - base);
      sum = fmaf(*cluster.map_shared_rank(&s->cl[g], r), f, sum);
      out = fmaf(*cluster.map_shared_rank(&s->co[g][c], r), f, out);
    }
    static_cast<T*>(a.o)[((int64_t)part.b * a.heads + part.head0 + g) * a.dim + c] = from_f32<T>(sum == 0.f ? 0.f : out / sum);
  }
  cluster.sync();  // no CTA leaves while another reads its shared memory
}

// ---- float32 -------------------------------------------------------------------

constexpr int kGroupF32 = 4;

__global__ void __launch_bounds__(kWarps * 32) attention_decode_f32(const DecodeArgs a) {
  constexpr int GC = kGroupF32, U = 4;  // U keys in flight per warp
  extern __shared__ float sbias[];
  __shared__ Partial<GC> sp;
  const Part<GC> p(a);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  load_bias(a, p, sbias);
  __syncthreads();
  const bool active = lane * 4 < a.dim;
  float4 q[GC];
  float o[GC][4], m[GC], l[GC];
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    m[g] = -CUDART_INF_F, l[g] = 0.f;
    o[g][0] = o[g][1] = o[g][2] = o[g][3] = 0.f;
    q[g] = g < p.n_g && active
               ? *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + p.b * a.q_batch + (p.head0 + g) * a.q_head + lane * 4)
               : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float* kp = static_cast<const float*>(a.k) + p.b * a.k_batch + p.kv_head * a.k_head + lane * 4;
  const float* vp = static_cast<const float*>(a.v) + p.b * a.v_batch + p.kv_head * a.v_head + lane * 4;
  const float c2 = a.scale * kLog2e;
  for (int key0 = p.first + warp * U; key0 < p.last; key0 += kWarps * U) {
    float4 kk[U], vv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      kk[u] = vv[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (active && key0 + u < p.last) {
        kk[u] = *reinterpret_cast<const float4*>(kp + (int64_t)(key0 + u) * a.k_row);
        vv[u] = *reinterpret_cast<const float4*>(vp + (int64_t)(key0 + u) * a.v_row);
      }
    }
#pragma unroll
    for (int g = 0; g < GC; ++g) {
      if (g >= p.n_g) break;
      float t[U], top = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        t[u] = q[g].x * kk[u].x + q[g].y * kk[u].y + q[g].z * kk[u].z + q[g].w * kk[u].w;
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) t[u] += __shfl_xor_sync(0xffffffffu, t[u], s);
        t[u] *= c2;
        if (a.table != nullptr && g < p.n_g && key0 + u < p.last)
          t[u] += sbias[g * (2 * a.span + 1) + clamp_dist(p.len - 1 - key0 - u, a.span)];
        if (key0 + u >= p.last) t[u] = -CUDART_INF_F;
        top = fmaxf(top, t[u]);
      }
      const float base = top == -CUDART_INF_F ? 0.f : top, fix = ex2(m[g] - base);
      m[g] = top;
      l[g] *= fix;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[g][c] *= fix;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e = ex2(t[u] - base);
        l[g] += e;
        o[g][0] = fmaf(e, vv[u].x, o[g][0]);
        o[g][1] = fmaf(e, vv[u].y, o[g][1]);
        o[g][2] = fmaf(e, vv[u].z, o[g][2]);
        o[g][3] = fmaf(e, vv[u].w, o[g][3]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < GC; ++g) {
    if (lane == 0) sp.m[warp][g] = m[g], sp.l[warp][g] = l[g];
#pragma unroll
    for (int c = 0; c < 4; ++c) sp.o[warp][g][lane * 4 + c] = o[g][c];
  }
  join<float>(a, p, &sp);
}

// ---- bf16 ----------------------------------------------------------------------

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint4 load16(const __nv_bfloat16* p, bool ok) {
  return ok ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ void copy16(uint32_t dst, const __nv_bfloat16* src, bool ok) {  // zeros where not ok
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 take16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
  return v;
}

constexpr int kGroupBf16 = 16;

constexpr int kStages = 3;
// bytes of a warp's stage: its lanes' 16-byte pieces of 16 keys and values
template <int DP>
constexpr int stage_bytes() { return 16 * DP * 2 * 2; }
template <int DP>
constexpr int decode_ring() {
  return std::max<int>(kWarps * kStages * stage_bytes<DP>(), (int)sizeof(Partial<kGroupBf16>));
}

template <int DP>
__global__ void __launch_bounds__(kWarps * 32, DP == 64 ? 3 : 2) attention_decode_bf16(const DecodeArgs a) {
  constexpr int GC = kGroupBf16, KC = DP / 32, VC = DP / 64;
  extern __shared__ __align__(16) uint8_t smem[];
  Partial<GC>* sp = reinterpret_cast<Partial<GC>*>(smem);  // in the ring's place, after it
  float* sbias = reinterpret_cast<float*>(smem + decode_ring<DP>());
  const Part<GC> p(a);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = lane >> 2, t = lane & 3;
  load_bias(a, p, sbias);
  const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(a.q) + p.b * a.q_batch + p.head0 * a.q_head;
  const __nv_bfloat16* kp = static_cast<const __nv_bfloat16*>(a.k) + p.b * a.k_batch + p.kv_head * a.k_head;
  const __nv_bfloat16* vp = static_cast<const __nv_bfloat16*>(a.v) + p.b * a.v_batch + p.kv_head * a.v_head;
  uint4 q[KC][2];  // rows n and n + 8
#pragma unroll
  for (int i = 0; i < KC; ++i)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      q[i][r] = load16(qp + (n + 8 * r) * a.q_head + i * 32 + t * 8, n + 8 * r < p.n_g && i * 32 + t * 8 < a.dim);
  __syncthreads();
  float o[VC][8][4] = {}, m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
  const float c2 = a.scale * kLog2e;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * kStages * stage_bytes<DP>() + lane * 16;
  // Pieces of a stage: K (h, i), then V (h, r).  The lane's first piece of the next tile to fetch;
  // columns past dim are zeros, rows past the slice too.
  const __nv_bfloat16* kf = kp + (int64_t)(p.first + warp * 16 + n) * a.k_row + t * 8;
  const __nv_bfloat16* vf = vp + (int64_t)(p.first + warp * 16 + 2 * t) * a.v_row + n * 8;
  const int64_t k8 = 8 * a.k_row, v8 = 8 * a.v_row;
  auto fetch = [&](int key0, int stage) {
    const uint32_t at = ring + stage * stage_bytes<DP>();
    if (key0 + 16 <= p.last && a.dim == DP) {
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        copy16(at + i * 512, kf + i * 32, true);
        copy16(at + (KC + i) * 512, kf + k8 + i * 32, true);
      }
#pragma unroll
      for (int h = 0; h < VC; ++h) {
        copy16(at + (2 * KC + h * 4) * 512, vf + h * 64, true);
        copy16(at + (2 * KC + h * 4 + 1) * 512, vf + a.v_row + h * 64, true);
        copy16(at + (2 * KC + h * 4 + 2) * 512, vf + v8 + h * 64, true);
        copy16(at + (2 * KC + h * 4 + 3) * 512, vf + v8 + a.v_row + h * 64, true);
      }
    } else if (key0 < p.last) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < KC; ++i) {
          const bool ok = key0 + h * 8 + n < p.last && i * 32 + t * 8 < a.dim;
          copy16(at + (h * KC + i) * 512, ok ? kf + h * k8 + i * 32 : kp, ok);
        }
#pragma unroll
      for (int h = 0; h < VC; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool ok = key0 + (r >> 1) * 8 + 2 * t + (r & 1) < p.last && h * 64 + n * 8 < a.dim;
          copy16(at + (2 * KC + h * 4 + r) * 512, ok ? vf + (r >> 1) * v8 + (r & 1) * a.v_row + h * 64 : vp, ok);
        }
    }
    kf += (int64_t)(kWarps * 16) * a.k_row, vf += (int64_t)(kWarps * 16) * a.v_row;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  constexpr int kStep = kWarps * 16;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(p.first + warp * 16 + i * kStep, i);
  int stage = 0;
  for (int key0 = p.first + warp * 16; key0 < p.last; key0 += kStep) {
    // the stage that was used last is free: every lane reads its own pieces only
    fetch(key0 + (kStages - 1) * kStep, stage == 0 ? kStages - 1 : stage - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    const uint32_t at = ring + stage * stage_bytes<DP>();
    if (++stage == kStages) stage = 0;
    float s[2][4] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const uint4 k = take16(at + (h * KC + i) * 512);
        mma_bf16(s[h], q[i][0].x, q[i][1].x, q[i][0].y, q[i][1].y, k.x, k.y);
        mma_bf16(s[h], q[i][0].z, q[i][1].z, q[i][0].w, q[i][1].w, k.z, k.w);
      }
    // s[h][2 r + e]: head n + 8 r, key key0 + 8 h + 2 t + e
    float top[2] = {-CUDART_INF_F, -CUDART_INF_F};
    if (a.table != nullptr || key0 + 16 > p.last) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int key = key0 + h * 8 + 2 * t + (c & 1), g = n + 8 * (c >> 1);
          float x = s[h][c] * c2;
          if (a.table != nullptr && g < p.n_g && key < p.last) x += sbias[g * (2 * a.span + 1) + clamp_dist(p.len - 1 - key, a.span)];
          s[h][c] = key < p.last ? x : -CUDART_INF_F;
        }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[h][c] *= c2;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) top[c >> 1] = fmaxf(top[c >> 1], s[h][c]);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
    }
    // the maximum in use follows the true one only past a distance of 2^8
    if (__any_sync(0xffffffffu, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float m_new = fmaxf(m[r], top[r]);
        const float fix = m_new == -CUDART_INF_F ? 1.f : exp2f(m[r] - m_new);
        m[r] = m_new;
        l[r] *= fix;
#pragma unroll
        for (int h = 0; h < VC; ++h)
#pragma unroll
          for (int j = 0; j < 8; ++j) o[h][j][2 * r] *= fix, o[h][j][2 * r + 1] *= fix;
      }
    }
    uint32_t hi[4], lo[4];  // P as the A operand: registers (h, r)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float base = m[r] == -CUDART_INF_F ? 0.f : m[r];
        const float e0 = ex2(s[h][2 * r] - base), e1 = ex2(s[h][2 * r + 1] - base);
        l[r] += e0 + e1;
        const uint32_t w = pack2(e0, e1);
        hi[h * 2 + r] = w;
        lo[h * 2 + r] = pack2(e0 - __uint_as_float(w << 16), e1 - __uint_as_float(w & 0xffff0000u));
      }
#pragma unroll
    for (int h = 0; h < VC; ++h) {
      uint4 v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = take16(at + (2 * KC + h * 4 + r) * 512);
      const uint32_t *r0 = &v[0].x, *r1 = &v[1].x, *r2 = &v[2].x, *r3 = &v[3].x;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
        const uint32_t b0 = __byte_perm(r0[j >> 1], r1[j >> 1], sel), b1 = __byte_perm(r2[j >> 1], r3[j >> 1], sel);
        mma_bf16(o[h][j], hi[0], hi[1], hi[2], hi[3], b0, b1);
        mma_bf16(o[h][j], lo[0], lo[1], lo[2], lo[3], b0, b1);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the rings are done with
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int g = n + 8 * r;
    if (g >= p.n_g) continue;
    if (t == 0) sp->m[warp][g] = m[r], sp->l[warp][g] = l[r];
#pragma unroll
    for (int h = 0; h < VC; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < 8; ++j) sp->o[warp][g][h * 64 + (2 * t + e) * 8 + j] = o[h][j][2 * r + e];
  }
  join<__nv_bfloat16>(a, p, sp);
}

// Slices per sequence: about four CTAs an SM (sequences differ in length, and
// slices even that out; half and twice as many were slower at the 48 caches
// above), none shorter than 64 keys of a full cache.
int split_count(int batch, int capacity, int ctas_per_sequence) {
  const int64_t want = std::min<int64_t>(cdiv(148 * 4, (int64_t)batch * ctas_per_sequence), cdiv(capacity, 64));
  int splits = 1;
  while (splits < want && splits < kMaxSplits) splits *= 2;
  return splits;
}

template <void (*Kernel)(const DecodeArgs)>
int launch(int group_cap, size_t smem, const DecodeArgs& a, int batch, cudaStream_t st) {
  static SmemAllowed allowed;
  static std::atomic<bool> wide[16];  // clusters of 16 are allowed on this device
  const int per_seq = a.kv_heads * (int)cdiv(a.heads / a.kv_heads, group_cap);
  const int splits = split_count(batch, a.capacity, per_seq);
  if (a.table != nullptr) smem += (size_t)std::min(group_cap, a.heads / a.kv_heads) * (2 * a.span + 1) * sizeof(float);
  if (int rc = allow_smem(Kernel, smem, allowed)) return rc;
  if (splits > 8) {
    int dev = 0;
    KF_CUDA_RET(cudaGetDevice(&dev));
    if (dev >= 16 || !wide[dev].load(std::memory_order_relaxed)) {
      KF_CUDA_RET(cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      if (dev < 16) wide[dev].store(true, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(splits, per_seq, batch), cfg.blockDim = dim3(kWarps * 32), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = splits > 1 ? 1 : 0;
  KF_CUDA_RET(cudaLaunchKernelEx(&cfg, Kernel, a));
  return KF_OK;
}

}  // namespace
}  // namespace kf

extern "C" int kf_attention_decode(const void* q, const void* k, const void* v, const int32_t* lengths, const void* table,
                                   const int32_t* buckets, void* o, const kf_decode_desc* d, void* stream) {
  using namespace kf;
  clear_error();
  const char* fn = "kf_attention_decode";
  KF_CHECK_ARG(d != nullptr, "%s: null descriptor", fn);
  KF_CHECK_ARG(d->heads >= 1 && d->kv_heads >= 1 && d->heads % d->kv_heads == 0, "%s: %d heads do not divide over %d key heads", fn,
               d->heads, d->kv_heads);
  KF_CHECK_ARG(d->heads <= 65535, "%s: %d heads", fn, d->heads);
  KF_CHECK_ARG(d->dim >= 8 && d->dim <= attn::kMaxDim && d->dim % 8 == 0, "%s: head width %d is not a multiple of 8 up to %d", fn,
               d->dim, attn::kMaxDim);
  KF_CHECK_ARG(d->dtype == KF_DTYPE_F32 || d->dtype == KF_DTYPE_BF16, "%s: types must be float32 or bfloat16", fn);
  KF_CHECK_ARG(d->batch >= 0 && d->batch <= 65535 && d->capacity >= 0, "%s: bad sizes", fn);
  KF_CHECK_ARG(d->span >= 0 && d->span <= attn::kMaxSpan, "%s: bias distances up to %d are outside [0, %d]", fn, d->span, attn::kMaxSpan);
  KF_CHECK_ARG(d->n_buckets >= 0 && d->n_buckets <= attn::kMaxBuckets, "%s: %d buckets exceed %d", fn, d->n_buckets, attn::kMaxBuckets);
  if (d->batch == 0) return KF_OK;
  KF_CHECK_ARG(q && o && lengths && (d->capacity == 0 || (k && v)), "%s: null argument", fn);
  KF_CHECK_ARG((table == nullptr) == (buckets == nullptr), "%s: the bias needs a table and buckets", fn);
  const int size = d->dtype == KF_DTYPE_F32 ? 4 : 2;
  KF_CHECK_ARG(aligned16({q, k, v, o}) &&
                   strides16(size, {{d->batch, d->q_batch}, {d->heads, d->q_head}, {d->batch, d->k_batch}, {d->capacity, d->k_row},
                                    {d->kv_heads, d->k_head}, {d->batch, d->v_batch}, {d->capacity, d->v_row}, {d->kv_heads, d->v_head}}),
               "%s: rows must start at multiples of 16 bytes", fn);
  if (int rc = bind_device(q)) return rc;
  DecodeArgs a{};
  a.q = q, a.k = k, a.v = v, a.lengths = lengths, a.table = table, a.buckets = buckets, a.o = o;
  a.q_batch = d->q_batch, a.q_head = d->q_head, a.k_batch = d->k_batch, a.k_row = d->k_row, a.k_head = d->k_head;
  a.v_batch = d->v_batch, a.v_row = d->v_row, a.v_head = d->v_head;
  a.capacity = d->capacity, a.heads = d->heads, a.kv_heads = d->kv_heads, a.dim = d->dim, a.span = d->span;
  a.n_buckets = d->n_buckets > 0 ? d->n_buckets : INT_MAX;
  a.table_bf16 = d->table_dtype == KF_DTYPE_BF16, a.scale = d->scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->dtype == KF_DTYPE_F32) return launch<attention_decode_f32>(kGroupF32, 0, a, d->batch, st);
  return d->dim <= 64 ? launch<attention_decode_bf16<64>>(kGroupBf16, decode_ring<64>(), a, d->batch, st)
                      : launch<attention_decode_bf16<128>>(kGroupBf16, decode_ring<128>(), a, d->batch, st);
}
