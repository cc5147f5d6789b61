// Attention over packed sequences on the CUDA cores: float32 forward and
// backward.
//
// A CTA of 16 x 16 threads owns 64 rows (queries, or keys in dK/dV) and walks
// over tiles of 64 of the other side.  A thread holds a 4 x 4 block of the
// scores and, of each output row, 4 x D/16 sums; operands are in shared memory
// with rows 4 floats longer than D, so that the 16-byte reads of 16 rows fall
// into different banks.  32 packed multiply-adds (two each) per eight 16-byte
// reads; tiles come by cp.async, the next K under the softmax and the next V under
// the next scores.  The FMA pipe and those reads bound it: 8 sequences of 1024,
// 12 heads of 64, both ways with a bias: forward 0.80 ms (32 TFLOP/s), dQ 1.16
// (33), dK dV 1.38 (37), where unpacked arithmetic and plain loads gave some 19.
// The tensor cores have no float32: three TF32 products for each of these would
// be the next step.  The backward runs dK/dV (rows = keys, sums over the heads that
// share a key head) and dQ (rows = queries) separately: both recompute the
// scores, and every sum has one order.
#include "attention.cuh"
#include "f32x2.cuh"
#include "umma.cuh"

namespace kf {
namespace {

using namespace attn;

constexpr int kTile = 64, kThreads = 256;

template <int D>
struct Ld {
  static constexpr int row = D + 4;
};
constexpr int kLdP = kTile + 4;

// Starts copying a tile of up to 64 rows into shared memory; rows past `n` and
// columns past `dim` become zeros without a read, so nothing outside the sequence
// enters a sum.
template <int D>
__device__ __forceinline__ void fetch_rows(float* dst, const Strided& s, int64_t row0, int n, int head, int dim) {
  const float* p = static_cast<const float*>(s.p) + head * s.head;
  const uint32_t to = umma::smem_u32(dst);
#pragma unroll
  for (int i = 0; i < kTile * D / 4 / kThreads; ++i) {
    const int e = (i * kThreads + threadIdx.x) * 4, r = e / D, c = e % D;
    const bool in = r < n && c < dim;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + (r * Ld<D>::row + c) * 4),
                 "l"(in ? p + (row0 + r) * s.row + c : p), "r"(in ? 16 : 0)
                 : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// All but the last `N` tiles that were started are there, for every thread.
template <int N>
__device__ __forceinline__ void rows_ready() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  __syncthreads();
}

__device__ __forceinline__ ulonglong2 load4(const float* p) { return *reinterpret_cast<const ulonglong2*>(p); }

// out[i][j] = a(row ty*4+i) . b(row tx+16j): sums over even and over odd columns, side by side
template <int D>
__device__ __forceinline__ void dot_rows(const float* a, const float* b, int ty, int tx, float (&out)[4][4]) {
  uint64_t acc[4][4] = {};
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    ulonglong2 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = load4(a + (ty * 4 + i) * Ld<D>::row + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = load4(b + (tx + 16 * j) * Ld<D>::row + d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fma2(x[i].y, y[j].y, fma2(x[i].x, y[j].x, acc[i][j]));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) out[i][j] = sum_of(acc[i][j]);
}

// acc[i][c] += sum_k p(row ty*4+i, k) m(row k, columns): pairs of the columns tx*4 + 64 q + (0..3)
template <int D>
__device__ __forceinline__ void dot_cols(const float* p, const float* m, int ty, int tx, uint64_t (&acc)[4][D / 32]) {
#pragma unroll 2
  for (int k = 0; k < kTile; k += 4) {
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(p + (ty * 4 + i) * kLdP + k);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int q = 0; q < D / 64; ++q) {
        const ulonglong2 y = load4(m + (k + e) * Ld<D>::row + tx * 4 + 64 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = e == 0 ? x[i].x : e == 1 ? x[i].y : e == 2 ? x[i].z : x[i].w;
          acc[i][2 * q] = fma2(pair(f), y.x, acc[i][2 * q]);
          acc[i][2 * q + 1] = fma2(pair(f), y.y, acc[i][2 * q + 1]);
        }
      }
  }
}

template <int D>
__device__ __forceinline__ void store_rows(float* out, int64_t row0, int n, int heads, int head, int dim, int ty, int tx,
                                           const uint64_t (&acc)[4][D / 32], const float (&mul)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    if (r >= n) continue;
    float* p = out + ((row0 + r) * heads + head) * dim;
#pragma unroll
    for (int q = 0; q < D / 64; ++q) {
      const int col = tx * 4 + 64 * q;
      const uint64_t f = pair(mul[i]);
      if (col < dim) *reinterpret_cast<ulonglong2*>(p + col) = make_ulonglong2(mul2(acc[i][2 * q], f), mul2(acc[i][2 * q + 1], f));
    }
  }
}

__device__ __forceinline__ float half_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float half_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int D>
__global__ void __launch_bounds__(kThreads) attention_fwd(const Args a) {
  extern __shared__ __align__(16) float smem[];
  float* sq = smem;
  float* sk = sq + kTile * Ld<D>::row;
  float* sv = sk + kTile * Ld<D>::row;
  float* sp = sv + kTile * Ld<D>::row;
  float* sbias = sp + kTile * kLdP;
  int tile;
  const Seq s = load_tile(a, blockIdx.x / a.heads, &tile);
  const int head = blockIdx.x % a.heads, kv_head = head / (a.heads / a.kv_heads);
  const int r0 = tile * kTile, n_rows = min(kTile, s.lq - r0), off = s.lk - s.lq;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int k_end = a.causal ? min(s.lk, r0 + n_rows + off) : s.lk;
  auto fetch = [&](float* to, const Strided& from, int k0) { fetch_rows<D>(to, from, s.k0 + k0, min(kTile, s.lk - k0), kv_head, a.dim); };
  fetch_rows<D>(sq, a.q, s.q0 + r0, n_rows, head, a.dim);
  if (k_end > 0) fetch(sk, a.k, 0), fetch(sv, a.v, 0);
  if (a.table != nullptr) expand_bias_f32(a, head, sbias, threadIdx.x, kThreads);
  float m[4], l[4];
  uint64_t o[4][D / 32];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -CUDART_INF_F, l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[i][c] = 0;
  }
  const float c2 = a.scale * kLog2e;
  for (int k0 = 0; k0 < k_end; k0 += kTile) {
    float t[4][4];
    rows_ready<1>();
    dot_rows<D>(sq, sk, ty, tx, t);
    __syncthreads();
    if (k0 + kTile < k_end) fetch(sk, a.k, k0 + kTile);  // arrives under what follows
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pos = r0 + ty * 4 + i + off;
      float top = -CUDART_INF_F;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + tx + 16 * j;
        float v = t[i][j] * c2;
        if (a.table != nullptr) v += sbias[clamp_dist(pos - key, a.span)];
        t[i][j] = (key < s.lk && (!a.causal || key <= pos)) ? v : -CUDART_INF_F;
        top = fmaxf(top, t[i][j]);
      }
      const float m_new = fmaxf(m[i], half_max(top));
      const float base = m_new == -CUDART_INF_F ? 0.f : m_new;  // no visible key yet
      const float fix = ex2(m[i] - base);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t[i][j] = ex2(t[i][j] - base);
        sum += t[i][j];
        sp[(ty * 4 + i) * kLdP + tx + 16 * j] = t[i][j];
      }
      l[i] = l[i] * fix + half_sum(sum);
      m[i] = m_new;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) o[i][c] = mul2(o[i][c], pair(fix));
    }
    // V of this tile (a warp reads back its own rows of P only)
    if (k0 + kTile < k_end)
      rows_ready<1>();
    else
      rows_ready<0>();
    dot_cols<D>(sp, sv, ty, tx, o);
    __syncthreads();
    if (k0 + kTile < k_end) fetch(sv, a.v, k0 + kTile);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");  // where there was no tile
  float inv[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    inv[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
    const int r = ty * 4 + i;
    if (a.lse != nullptr && tx == 0 && r < n_rows)
      store_lse(a, head * a.tq + s.q0 + r0 + r, m[i], l[i]);
  }
  store_rows<D>(static_cast<float*>(a.o), s.q0 + r0, n_rows, a.heads, head, a.dim, ty, tx, o, inv);
}

// delta[h][i] = dO_i . O_i: one warp per (token, head).
__global__ void __launch_bounds__(256) attention_delta(const Args a) {
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= a.tq * a.heads) return;
  const int64_t tok = i / a.heads;
  const int head = (int)(i - tok * a.heads), lane = threadIdx.x & 31;
  const float* o = static_cast<const float*>(a.o) + i * a.dim;
  const float* g = static_cast<const float*>(a.dout.p) + tok * a.dout.row + head * a.dout.head;
  float v = 0.f;
  for (int c = lane; c < a.dim; c += 32) v = fmaf(o[c], g[c], v);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  if (lane == 0) a.delta[head * a.tq + tok] = v;
}

// Rows = queries: dQ = scale dS K, and the bias gradient's sums by distance.
template <int D>
__global__ void __launch_bounds__(kThreads) attention_dq(const Args a) {
  extern __shared__ __align__(16) float smem[];
  float* sq = smem;
  float* sg = sq + kTile * Ld<D>::row;
  float* sk = sg + kTile * Ld<D>::row;
  float* sv = sk + kTile * Ld<D>::row;
  float* sp = sv + kTile * Ld<D>::row;
  float* sbias = sp + kTile * kLdP;
  float* ssum = sbias + 2 * a.span + 1;  // gradient sums by clamped distance
  int tile;
  const Seq s = load_tile(a, blockIdx.x / a.heads, &tile);
  const int head = blockIdx.x % a.heads, kv_head = head / (a.heads / a.kv_heads);
  const int r0 = tile * kTile, n_rows = min(kTile, s.lq - r0), off = s.lk - s.lq;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int k_end = a.causal ? min(s.lk, r0 + n_rows + off) : s.lk;
  auto fetch = [&](float* to, const Strided& from, int k0) { fetch_rows<D>(to, from, s.k0 + k0, min(kTile, s.lk - k0), kv_head, a.dim); };
  fetch_rows<D>(sq, a.q, s.q0 + r0, n_rows, head, a.dim);
  fetch_rows<D>(sg, a.dout, s.q0 + r0, n_rows, head, a.dim);
  if (k_end > 0) fetch(sv, a.v, 0), fetch(sk, a.k, 0);
  if (a.table != nullptr) {
    expand_bias_f32(a, head, sbias, threadIdx.x, kThreads);
    for (int i = threadIdx.x; i < 2 * a.span + 1; i += kThreads) ssum[i] = 0.f;
  }
  float lse[4], rest[4], delta[4], far[2] = {0.f, 0.f};  // far: sums beyond the span
  uint64_t dq[4][D / 32];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    lse[i] = r < n_rows ? a.lse[head * a.tq + s.q0 + r0 + r] : 0.f;
    rest[i] = r < n_rows ? load_lse_rest(a, head * a.tq + s.q0 + r0 + r) : 0.f;
    delta[i] = r < n_rows ? a.delta[head * a.tq + s.q0 + r0 + r] : 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dq[i][c] = 0;
  }
  const float c2 = a.scale * kLog2e;
  for (int k0 = 0; k0 < k_end; k0 += kTile) {
    float t[4][4], dp[4][4];
    rows_ready<0>();
    dot_rows<D>(sg, sv, ty, tx, dp);
    dot_rows<D>(sq, sk, ty, tx, t);
    __syncthreads();
    if (k0 + kTile < k_end) fetch(sv, a.v, k0 + kTile);  // arrives under what follows
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pos = r0 + ty * 4 + i + off;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + tx + 16 * j;
        float v = t[i][j] * c2;
        if (a.table != nullptr) v += sbias[clamp_dist(pos - key, a.span)];
        const bool visible = ty * 4 + i < n_rows && key < s.lk && (!a.causal || key <= pos) && !one_key(a, s, pos);
        sp[(ty * 4 + i) * kLdP + tx + 16 * j] = visible ? ex2((v - lse[i]) - rest[i]) * (dp[i][j] - delta[i]) : 0.f;
      }
    }
    __syncwarp();
    dot_cols<D>(sp, sk, ty, tx, dq);
    if (a.dist_part != nullptr) {
      // thread d sums the diagonal row - column = d - 63 of dS; those beyond the span stay with it until the end
      __syncthreads();
      float sum = 0.f;
      const int d = (int)threadIdx.x - (kTile - 1), dist = r0 + off - k0 + d;
      if (threadIdx.x < 2 * kTile - 1) {
        const int first = max(0, d), last = min(kTile, kTile + d);
#pragma unroll 8
        for (int r = first; r < last; ++r) sum += sp[r * kLdP + r - d];
        if (dist <= -a.span)
          far[0] += sum;
        else if (dist >= a.span)
          far[1] += sum;
        else
          ssum[dist + a.span] += sum;
      }
    }
    __syncthreads();
    if (k0 + kTile < k_end) fetch(sk, a.k, k0 + kTile);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");  // where there was no tile
  const float mul[4] = {a.scale, a.scale, a.scale, a.scale};
  store_rows<D>(static_cast<float*>(a.dq), s.q0 + r0, n_rows, a.heads, head, a.dim, ty, tx, dq, mul);
  if (a.dist_part != nullptr) {
    __syncthreads();
    float* out = a.dist_part + (int64_t)blockIdx.x * (2 * a.span + 1);
    for (int e = threadIdx.x; e < 2 * a.span + 1; e += kThreads)
      if (e > 0 && e < 2 * a.span) out[e] = ssum[e];
    sp[threadIdx.x] = far[0], sp[kThreads + threadIdx.x] = far[1];
    __syncthreads();
    const int side = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (side < 2) {
      float sum = 0.f;
      for (int i = lane; i < 2 * kTile; i += 32) sum += sp[side * kThreads + i];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) out[side * 2 * a.span] = sum;
    }
  }
}

// Rows = keys: dV = P^T dO and dK = scale dS^T Q, summed over the heads of the group.
template <int D>
__global__ void __launch_bounds__(kThreads) attention_dkdv(const Args a) {
  extern __shared__ __align__(16) float smem[];
  float* sk = smem;
  float* sv = sk + kTile * Ld<D>::row;
  float* sq = sv + kTile * Ld<D>::row;
  float* sg = sq + kTile * Ld<D>::row;
  float* sp = sg + kTile * Ld<D>::row;
  float* sds = sp + kTile * kLdP;
  float* slse = sds + kTile * kLdP;
  float* srest = slse + kTile;
  float* sdelta = srest + kTile;
  float* sbias = sdelta + kTile;
  int tile;
  const Seq s = load_tile(a, blockIdx.x / a.kv_heads, &tile);
  const int kv_head = blockIdx.x % a.kv_heads, group = a.heads / a.kv_heads;
  const int r0 = tile * kTile, n_rows = min(kTile, s.lk - r0), off = s.lk - s.lq;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  fetch_rows<D>(sk, a.k, s.k0 + r0, n_rows, kv_head, a.dim);
  fetch_rows<D>(sv, a.v, s.k0 + r0, n_rows, kv_head, a.dim);
  uint64_t dk[4][D / 32], dv[4][D / 32];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dk[i][c] = dv[i][c] = 0;
  const int q_first = a.causal ? max(0, r0 - off) / kTile * kTile : 0;  // earlier queries see none of these keys
  const float c2 = a.scale * kLog2e;
  for (int head = kv_head * group; head < (kv_head + 1) * group; ++head) {
    __syncthreads();
    if (a.table != nullptr) expand_bias_f32(a, head, sbias, threadIdx.x, kThreads);
    for (int q0 = q_first; q0 < s.lq; q0 += kTile) {
      const int n_q = min(kTile, s.lq - q0);
      __syncthreads();
      fetch_rows<D>(sq, a.q, s.q0 + q0, n_q, head, a.dim);
      fetch_rows<D>(sg, a.dout, s.q0 + q0, n_q, head, a.dim);
      if (threadIdx.x < kTile) {
        const bool in = (int)threadIdx.x < n_q;
        slse[threadIdx.x] = in ? a.lse[head * a.tq + s.q0 + q0 + threadIdx.x] : 0.f;
        srest[threadIdx.x] = in ? load_lse_rest(a, head * a.tq + s.q0 + q0 + threadIdx.x) : 0.f;
        sdelta[threadIdx.x] = in ? a.delta[head * a.tq + s.q0 + q0 + threadIdx.x] : 0.f;
      }
      rows_ready<0>();
      float t[4][4], dp[4][4];
      dot_rows<D>(sk, sq, ty, tx, t);
      dot_rows<D>(sv, sg, ty, tx, dp);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = r0 + ty * 4 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = tx + 16 * j, pos = q0 + c + off;
          float v = t[i][j] * c2;
          if (a.table != nullptr) v += sbias[clamp_dist(pos - key, a.span)];
          const bool visible = c < n_q && key < s.lk && (!a.causal || key <= pos);
          const float p = visible ? ex2((v - slse[c]) - srest[c]) : 0.f;
          sp[(ty * 4 + i) * kLdP + c] = p;
          sds[(ty * 4 + i) * kLdP + c] = visible && !one_key(a, s, pos) ? p * (dp[i][j] - sdelta[c]) : 0.f;
        }
      }
      __syncwarp();
      dot_cols<D>(sp, sg, ty, tx, dv);
      dot_cols<D>(sds, sq, ty, tx, dk);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");  // where there was no tile
  const float one[4] = {1.f, 1.f, 1.f, 1.f}, mul[4] = {a.scale, a.scale, a.scale, a.scale};
  store_rows<D>(static_cast<float*>(a.dv), s.k0 + r0, n_rows, a.kv_heads, kv_head, a.dim, ty, tx, dv, one);
  store_rows<D>(static_cast<float*>(a.dk), s.k0 + r0, n_rows, a.kv_heads, kv_head, a.dim, ty, tx, dk, mul);
}

template <void (*Kernel)(const Args)>
int run(unsigned grid, size_t floats, const Args& a, cudaStream_t st, const char* what) {
  static SmemAllowed allowed;
  if (int rc = allow_smem(Kernel, floats * sizeof(float), allowed)) return rc;
  Kernel<<<grid, kThreads, floats * sizeof(float), st>>>(a);
  return check_launch(what);
}

template <int D>
int fwd(const Args& a, int n_tiles, cudaStream_t st) {
  const size_t bias = a.table != nullptr ? 2 * a.span + 1 : 0;
  return run<attention_fwd<D>>((unsigned)n_tiles * a.heads, 3 * kTile * Ld<D>::row + kTile * kLdP + bias, a, st, "kf_attention_fwd");
}

template <int D>
int bwd(const Args& a0, const Tile* k_tiles, int n_q, int n_k, cudaStream_t st) {
  Args a = a0;
  const size_t bias = a.table != nullptr ? 2 * a.span + 1 : 0;
  if (a.tq > 0) {
    attention_delta<<<(unsigned)cdiv(a.tq * a.heads, 8), 256, 0, st>>>(a);
    if (int rc = check_launch("kf_attention_bwd")) return rc;
  }
  if (n_q > 0)
    if (int rc = run<attention_dq<D>>((unsigned)n_q * a.heads, 4 * kTile * Ld<D>::row + kTile * kLdP + 2 * bias, a, st, "kf_attention_bwd"))
      return rc;
  a.tiles = k_tiles;
  if (n_k > 0)
    return run<attention_dkdv<D>>((unsigned)n_k * a.kv_heads, 4 * kTile * Ld<D>::row + 2 * kTile * kLdP + 3 * kTile + bias, a, st,
               "kf_attention_bwd");
  return KF_OK;
}

}  // namespace

namespace attn {
int fwd_f32(const Args& a, int n_tiles, cudaStream_t st) {
  return a.dim <= 64 ? fwd<64>(a, n_tiles, st) : fwd<128>(a, n_tiles, st);
}
int bwd_f32(const Args& a, const Tile* k_tiles, int n_q, int n_k, cudaStream_t st) {
  return a.dim <= 64 ? bwd<64>(a, k_tiles, n_q, n_k, st) : bwd<128>(a, k_tiles, n_q, n_k, st);
}
}  // namespace attn
}  // namespace kf
