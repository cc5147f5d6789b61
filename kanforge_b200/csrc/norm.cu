// Residual norm: the join between two blocks of a transformer in one pass over
// its rows,
//   u = N_b(branch) w_b + s_b   (or the branch itself),
//   y = alpha x + gate * u,     h = N(y) w + s,
// with N(v) = (v - mean) / sqrt(var + eps) ("layer") or v / sqrt(mean v^2 + eps)
// ("rms"), and its backward
//   g = dy + rstd (a - [mean a] - yhat mean(a yhat)),  a = dh w
//   dx = alpha g, du = gate g, dgate = g u, dbranch = N_b'(du w_b),
//   dw = sum dh yhat, ds = sum dh, dw_b = sum du bhat, ds_b = sum du.
//
// Both are bound by HBM: the forward reads x and the branch and writes y and h,
// the backward reads dy, dh, x and the branch and writes dx and dbranch.  A row
// stays in the registers of the W warps that own it; its sums cross lanes by
// shuffles and warps by one exchange in shared memory.  Everything between the
// loads and the stores is float32.
#include "common.cuh"

namespace kf {
namespace {

constexpr int kMaxWidth = 8192;
constexpr int kParamGrads = 5;  // dw, ds, dgate, dw_b, ds_b

struct RowArgs {
  const void* x;
  const void* branch;
  const void* gate;  // per token (rows, width) in the branch's type, or per channel in the parameters' type
  const void* w;
  const void* s;
  const void* bw;
  const void* bs;
  void* y;
  void* h;
  float4* stats;  // mean and rstd of y, mean and rstd of the branch
  int64_t rows;
  int width;
  float alpha, eps;
  bool layer, branch_norm, gate_token, param_bf16;
  int warps;  // per row
};

struct GradArgs {
  RowArgs f;
  const void* dy;  // may be null: no gradient reached y
  const void* dh;  // likewise
  void* dx;
  void* dbranch;
  void* dgate;  // per token only; the other parameter gradients go to `part`
  float* part;  // (gridDim.x, 5, width)
};

// Elements of a row owned by a lane, in V chunks of 8.  Aligned rows (width a
// multiple of 8) are read in 16-byte vectors; other rows element by element,
// lanes on neighbouring elements.
template <bool VEC>
__device__ __forceinline__ int elem(int c, int k, int warps, int wl) {
  return VEC ? (c * warps * 32 + wl) * 8 + k : (c * 8 + k) * warps * 32 + wl;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint4 a;
  uint32_t* w = &a.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  *reinterpret_cast<uint4*>(p) = a;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_chunk(const T* row, int width, int c, int warps, int wl, float (&v)[8]) {
  if (VEC) {
    const int e = elem<true>(c, 0, warps, wl);
    if (e < width) {
      load8(row + e, v);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = 0.f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int e = elem<false>(c, k, warps, wl);
      v[k] = e < width ? to_f32<T>(row[e]) : 0.f;
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_chunk(T* row, int width, int c, int warps, int wl, const float (&v)[8]) {
  if (VEC) {
    const int e = elem<true>(c, 0, warps, wl);
    if (e < width) store8(row + e, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int e = elem<false>(c, k, warps, wl);
      if (e < width) row[e] = from_f32<T>(v[k]);
    }
  }
}

template <bool VEC>
__device__ __forceinline__ void load_param(const void* p, bool bf16, int width, int c, int warps, int wl, float (&v)[8]) {
  if (bf16)
    load_chunk<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16*>(p), width, c, warps, wl, v);
  else
    load_chunk<float, VEC>(static_cast<const float*>(p), width, c, warps, wl, v);
}

template <bool VEC>
__device__ __forceinline__ bool owned(int c, int k, int width, int warps, int wl) {
  return elem<VEC>(c, k, warps, wl) < width;
}

// u of one chunk: the branch, normed by st.z and st.w where that is asked for.
template <bool VEC>
__device__ __forceinline__ void branch_value(const RowArgs& a, const float (&br)[8], const float4& st, int c, int wl, float (&u)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] = br[k];
  if (!a.branch_norm) return;
  float p[8];
  load_param<VEC>(a.bw, a.param_bf16, a.width, c, a.warps, wl, p);
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] = (u[k] - st.z) * st.w * p[k];
  if (a.bs == nullptr) return;
  load_param<VEC>(a.bs, a.param_bf16, a.width, c, a.warps, wl, p);
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] += p[k];
}

template <typename TB, bool VEC>
__device__ __forceinline__ void load_gate(const RowArgs& a, int64_t off, int c, int wl, float (&t)[8]) {
  if (a.gate_token)
    load_chunk<TB, VEC>(static_cast<const TB*>(a.gate) + off, a.width, c, a.warps, wl, t);
  else
    load_param<VEC>(a.gate, a.param_bf16, a.width, c, a.warps, wl, t);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The warps that share a row: sums over them, in warp order, so every lane
// of every warp gets the same bits.  Two exchange buffers alternate, so one
// barrier per exchange is enough.
struct RowGroup {
  float* buf;  // 2 x warps x 3 floats
  int warps, warp, lane, barrier;
  int phase;

  __device__ __forceinline__ const float* exchange(float a, float b, float c) {
    float* p = buf + phase * warps * 3;
    phase ^= 1;
    if (lane == 0) p[warp * 3] = a, p[warp * 3 + 1] = b, p[warp * 3 + 2] = c;
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
    return p;
  }

  __device__ __forceinline__ void sum2(float& a, float& b) {
    a = warp_sum(a), b = warp_sum(b);
    if (warps == 1) return;
    const float* p = exchange(a, b, 0.f);
    a = b = 0.f;
    for (int w = 0; w < warps; ++w) a += p[w * 3], b += p[w * 3 + 1];
  }

  // Mean and reciprocal standard deviation of the group's row.  "layer": the
  // squares are taken about the warp's own mean and the warps' moments merged,
  // so a large mean costs no digits and one exchange is enough.
  template <int V, bool VEC>
  __device__ __forceinline__ float2 moments(const float (&v)[V][8], int width, int wl, float eps, bool layer) {
    float n = 0.f, sum = 0.f, sq = 0.f;
    if (!layer) {
#pragma unroll
      for (int c = 0; c < V; ++c)
#pragma unroll
        for (int k = 0; k < 8; ++k) sq = fmaf(v[c][k], v[c][k], sq);  // elements past the width are 0
      sum2(sq, sum);
      return make_float2(0.f, 1.f / sqrtf(sq / width + eps));
    }
#pragma unroll
    for (int c = 0; c < V; ++c)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        sum += v[c][k];
        n += owned<VEC>(c, k, width, warps, wl) ? 1.f : 0.f;
      }
    sum = warp_sum(sum), n = warp_sum(n);
    float mean = n > 0.f ? sum / n : 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float d = owned<VEC>(c, k, width, warps, wl) ? v[c][k] - mean : 0.f;
        sq = fmaf(d, d, sq);
      }
    sq = warp_sum(sq);
    if (warps > 1) {
      const float* p = exchange(n, sum, sq);
      float total = 0.f;
      for (int w = 0; w < warps; ++w) total += p[w * 3 + 1];
      mean = total / width;
      sq = 0.f;
      for (int w = 0; w < warps; ++w) {
        const float nw = p[w * 3], d = nw > 0.f ? p[w * 3 + 1] / nw - mean : 0.f;
        sq += p[w * 3 + 2] + nw * d * d;
      }
    }
    return make_float2(mean, 1.f / sqrtf(sq / width + eps));
  }
};

template <int V, bool VEC, typename TX, typename TB>
__global__ void __launch_bounds__(512) residual_norm_fwd(const RowArgs a) {
  extern __shared__ float exch[];
  const int lane = threadIdx.x & 31, warp_id = threadIdx.x >> 5, group = warp_id / a.warps;
  RowGroup g{exch + group * 2 * a.warps * 3, a.warps, warp_id - group * a.warps, lane, 1 + group, 0};
  const int wl = g.warp * 32 + lane;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / 32 / a.warps) + group;
  if (row >= a.rows) return;
  float y[V][8];
#pragma unroll
  for (int c = 0; c < V; ++c)
    load_chunk<TX, VEC>(static_cast<const TX*>(a.x) + row * a.width, a.width, c, a.warps, wl, y[c]);
  float2 sb = make_float2(0.f, 1.f);
  if (a.branch != nullptr) {
    float u[V][8];
#pragma unroll
    for (int c = 0; c < V; ++c)
      load_chunk<TB, VEC>(static_cast<const TB*>(a.branch) + row * a.width, a.width, c, a.warps, wl, u[c]);
    if (a.branch_norm) {
      sb = g.moments<V, VEC>(u, a.width, wl, a.eps, a.layer);
#pragma unroll
      for (int c = 0; c < V; ++c) branch_value<VEC>(a, u[c], make_float4(0.f, 0.f, sb.x, sb.y), c, wl, u[c]);
    }
#pragma unroll
    for (int c = 0; c < V; ++c) {
      if (a.gate != nullptr) {
        float t[8];
        load_gate<TB, VEC>(a, row * a.width, c, wl, t);
#pragma unroll
        for (int k = 0; k < 8; ++k) u[c][k] *= t[k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)  // past the width: a row's shift must not leak into the sums
        y[c][k] = owned<VEC>(c, k, a.width, a.warps, wl) ? fmaf(a.alpha, y[c][k], u[c][k]) : 0.f;
      store_chunk<TX, VEC>(static_cast<TX*>(a.y) + row * a.width, a.width, c, a.warps, wl, y[c]);
    }
  }
  const float2 sy = g.moments<V, VEC>(y, a.width, wl, a.eps, a.layer);
#pragma unroll
  for (int c = 0; c < V; ++c) {
    float w[8], s[8], o[8];
    load_param<VEC>(a.w, a.param_bf16, a.width, c, a.warps, wl, w);
    if (a.s != nullptr) load_param<VEC>(a.s, a.param_bf16, a.width, c, a.warps, wl, s);
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = (y[c][k] - sy.x) * sy.y * w[k] + (a.s != nullptr ? s[k] : 0.f);
    store_chunk<TB, VEC>(static_cast<TB*>(a.h) + row * a.width, a.width, c, a.warps, wl, o);
  }
  if (a.stats != nullptr && wl == 0) a.stats[row] = make_float4(sy.x, sy.y, sb.x, sb.y);
}

// One CTA walks over rows blockIdx.x * groups + group, + gridDim.x * groups, ...
// The parameter gradients' column sums stay with the lane that owns the
// columns: in registers while a lane owns 8 columns (V = 1, widths up to 4096),
// in shared memory above, then one partial sum per CTA in `part`.
template <int V, bool VEC, typename TX, typename TB>
__global__ void __launch_bounds__(512) residual_norm_bwd(const GradArgs p) {
  extern __shared__ float smem[];
  const RowArgs& a = p.f;
  const int lane = threadIdx.x & 31, warp_id = threadIdx.x >> 5, group = warp_id / a.warps;
  const int groups = blockDim.x / 32 / a.warps;
  float* sums = smem;  // (5, width)
  RowGroup g{smem + kParamGrads * a.width + group * 2 * a.warps * 3, a.warps, warp_id - group * a.warps, lane, 1 + group, 0};
  const int wl = g.warp * 32 + lane;
  constexpr bool REGS = V == 1;
  float acc[REGS ? kParamGrads : 1][8];
#pragma unroll
  for (int j = 0; j < (REGS ? kParamGrads : 1); ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[j][k] = 0.f;
  for (int i = threadIdx.x; i < kParamGrads * a.width; i += blockDim.x) sums[i] = 0.f;
  __syncthreads();
  const float inv = 1.f / a.width;

  auto add = [&](int j, int c, const float(&v)[8]) {
    if (REGS) {
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[REGS ? j : 0][k] += v[k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = elem<VEC>(c, k, a.warps, wl);
        if (e < a.width) sums[j * a.width + e] += v[k];
      }
    }
  };

  for (int64_t row = (int64_t)blockIdx.x * groups + group; row < a.rows; row += (int64_t)gridDim.x * groups) {
    const int64_t off = row * a.width;
    const float4 st = a.stats[row];
    float hat[V][8], dh[V][8], gr[V][8], br[V][8];
#pragma unroll
    for (int c = 0; c < V; ++c) {
      load_chunk<TX, VEC>(static_cast<const TX*>(a.x) + off, a.width, c, a.warps, wl, hat[c]);
      if (p.dh != nullptr) {
        load_chunk<TB, VEC>(static_cast<const TB*>(p.dh) + off, a.width, c, a.warps, wl, dh[c]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) dh[c][k] = 0.f;
      }
      if (p.dy != nullptr) {
        load_chunk<TX, VEC>(static_cast<const TX*>(p.dy) + off, a.width, c, a.warps, wl, gr[c]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) gr[c][k] = 0.f;
      }
      if (a.branch != nullptr)
        load_chunk<TB, VEC>(static_cast<const TB*>(a.branch) + off, a.width, c, a.warps, wl, br[c]);
    }
    // y again, from x and the branch and not from its rounded copy: as many bytes to read, and no rounding in yhat
#pragma unroll
    for (int c = 0; c < V; ++c) {
      if (a.branch != nullptr) {
        float u[8], t[8];
        branch_value<VEC>(a, br[c], st, c, wl, u);
        if (a.gate != nullptr) {
          load_gate<TB, VEC>(a, off, c, wl, t);
#pragma unroll
          for (int k = 0; k < 8; ++k) u[k] *= t[k];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) hat[c][k] = fmaf(a.alpha, hat[c][k], u[k]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) hat[c][k] = owned<VEC>(c, k, a.width, a.warps, wl) ? (hat[c][k] - st.x) * st.y : 0.f;
    }
    float m1 = 0.f, m2 = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      float w[8], t[8];
      load_param<VEC>(a.w, a.param_bf16, a.width, c, a.warps, wl, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        t[k] = dh[c][k] * hat[c][k];
      }
      add(0, c, t);
      add(1, c, dh[c]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        dh[c][k] *= w[k];
        m1 += dh[c][k];
        m2 = fmaf(dh[c][k], hat[c][k], m2);
      }
    }
    g.sum2(m1, m2);
    m1 = a.layer ? m1 * inv : 0.f;
    m2 *= inv;
#pragma unroll
    for (int c = 0; c < V; ++c) {
#pragma unroll
      for (int k = 0; k < 8; ++k) gr[c][k] += st.y * (dh[c][k] - m1 - hat[c][k] * m2);
      float t[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = a.alpha * gr[c][k];
      store_chunk<TX, VEC>(static_cast<TX*>(p.dx) + off, a.width, c, a.warps, wl, t);
    }
    if (a.branch == nullptr) continue;
    // from here dh holds du w_b and hat the normalised branch
    m1 = m2 = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      float u[8], w[8], t[8];
      branch_value<VEC>(a, br[c], st, c, wl, u);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        hat[c][k] = (br[c][k] - st.z) * st.w;
        w[k] = 1.f;
      }
      if (a.branch_norm) load_param<VEC>(a.bw, a.param_bf16, a.width, c, a.warps, wl, w);
      if (a.gate != nullptr) {
        load_gate<TB, VEC>(a, off, c, wl, t);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          u[k] *= gr[c][k];
          gr[c][k] *= t[k];
        }
        if (a.gate_token)
          store_chunk<TB, VEC>(static_cast<TB*>(p.dgate) + off, a.width, c, a.warps, wl, u);
        else
          add(2, c, u);
      }
      if (a.branch_norm) {
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = gr[c][k] * hat[c][k];
        add(3, c, t);
        add(4, c, gr[c]);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        dh[c][k] = gr[c][k] * w[k];
        m1 += dh[c][k];
        m2 = fmaf(dh[c][k], hat[c][k], m2);
      }
    }
    if (a.branch_norm) {
      g.sum2(m1, m2);
      m1 = a.layer ? m1 * inv : 0.f;
      m2 *= inv;
#pragma unroll
      for (int c = 0; c < V; ++c)
#pragma unroll
        for (int k = 0; k < 8; ++k) dh[c][k] = st.w * (dh[c][k] - m1 - hat[c][k] * m2);
    }
#pragma unroll
    for (int c = 0; c < V; ++c)
      store_chunk<TB, VEC>(static_cast<TB*>(p.dbranch) + off, a.width, c, a.warps, wl, dh[c]);
  }

  // the groups' sums join in group order
  if (REGS) {
    for (int r = 0; r < groups; ++r) {
      __syncthreads();
      if (r == group) {
#pragma unroll
        for (int j = 0; j < kParamGrads; ++j)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int e = elem<VEC>(0, k, a.warps, wl);
            if (e < a.width) sums[j * a.width + e] += acc[REGS ? j : 0][k];
          }
      }
    }
  }
  __syncthreads();
  float* out = p.part + (int64_t)blockIdx.x * kParamGrads * a.width;
  for (int i = threadIdx.x; i < kParamGrads * a.width; i += blockDim.x) out[i] = sums[i];
}

struct ParamOut {
  void* out[kParamGrads];  // null: not wanted
};

// Column sums of the CTAs' partial sums, in a fixed order: 32 columns by 8
// slices of the CTAs, slices joined in order.
__global__ void __launch_bounds__(256) residual_norm_params(const float* part, int n_part, int width, ParamOut o, bool bf16) {
  __shared__ float s[8][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5, j = blockIdx.y;
  if (o.out[j] == nullptr) return;
  float v = 0.f;
  if (col < width)
    for (int i = slice; i < n_part; i += 8) v += part[((int64_t)i * kParamGrads + j) * width + col];
  s[slice][threadIdx.x & 31] = v;
  __syncthreads();
  if (slice != 0 || col >= width) return;
  v = 0.f;
  for (int i = 0; i < 8; ++i) v += s[i][threadIdx.x];
  if (bf16)
    static_cast<__nv_bfloat16*>(o.out[j])[col] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(o.out[j])[col] = v;
}

bool rows_aligned(std::initializer_list<const void*> ps, int width) {
  if (width % 8) return false;
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}


// CTAs of the backward: two per SM, fewer when there are fewer rows than CTAs.
int bwd_ctas(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>(rows, 296)); }

template <int V, bool VEC, typename TX, typename TB>
int launch_fwd(RowArgs a, int groups, cudaStream_t s) {
  const size_t smem = (size_t)groups * 2 * a.warps * 3 * sizeof(float);
  residual_norm_fwd<V, VEC, TX, TB><<<(unsigned)cdiv(a.rows, groups), groups * a.warps * 32, smem, s>>>(a);
  return check_launch("kf_residual_norm_fwd");
}

template <int V, bool VEC, typename TX, typename TB>
int launch_bwd(GradArgs p, int groups, int ctas, cudaStream_t s) {
  const size_t smem = (size_t)(kParamGrads * p.f.width + groups * 2 * p.f.warps * 3) * sizeof(float);
  auto* k = residual_norm_bwd<V, VEC, TX, TB>;
  KF_CUDA_RET(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  k<<<ctas, groups * p.f.warps * 32, smem, s>>>(p);
  return check_launch("kf_residual_norm_bwd");
}

template <bool VEC, typename TX, typename TB>
int dispatch_fwd(RowArgs a, cudaStream_t s) {
  // 8 elements a lane while a row fits 16 warps (widths to 4096), 16 above
  const int per_warp = a.width <= 4096 ? 256 : 512;
  a.warps = (int)cdiv(a.width, per_warp);
  const int groups = std::max(1, 8 / a.warps);
  return per_warp == 256 ? launch_fwd<1, VEC, TX, TB>(a, groups, s) : launch_fwd<2, VEC, TX, TB>(a, groups, s);
}

template <bool VEC, typename TX, typename TB>
int dispatch_bwd(GradArgs p, int ctas, cudaStream_t s) {
  const int per_warp = p.f.width <= 4096 ? 256 : 512;
  p.f.warps = (int)cdiv(p.f.width, per_warp);
  const int groups = std::max(1, 8 / p.f.warps);
  return per_warp == 256 ? launch_bwd<1, VEC, TX, TB>(p, groups, ctas, s) : launch_bwd<2, VEC, TX, TB>(p, groups, ctas, s);
}

int check_common(const char* fn, const kf_residual_norm_desc* d, const void* x, const void* w, int64_t rows) {
  KF_CHECK_ARG(d != nullptr && (x != nullptr || rows == 0) && w != nullptr, "%s: null argument", fn);
  KF_CHECK_ARG(rows >= 0, "%s: %lld rows", fn, (long long)rows);
  KF_CHECK_ARG(d->width >= 1 && d->width <= kMaxWidth, "%s: rows of %d elements are outside [1, %d]", fn, d->width, kMaxWidth);
  KF_CHECK_ARG((d->x_dtype == KF_DTYPE_F32 || d->x_dtype == KF_DTYPE_BF16) &&
                   (d->branch_dtype == KF_DTYPE_F32 || d->branch_dtype == KF_DTYPE_BF16) &&
                   (d->param_dtype == KF_DTYPE_F32 || d->param_dtype == KF_DTYPE_BF16),
               "%s: types must be float32 or bfloat16", fn);
  KF_CHECK_ARG(!(d->x_dtype == KF_DTYPE_BF16 && d->branch_dtype == KF_DTYPE_F32), "%s: a bfloat16 sum takes no float32 branch", fn);
  KF_CHECK_ARG(d->eps >= 0.f, "%s: eps is negative", fn);
  return KF_OK;
}

RowArgs row_args(const kf_residual_norm_desc* d, int64_t rows) {
  RowArgs a{};
  a.rows = rows, a.width = d->width, a.alpha = d->residual_scale, a.eps = d->eps;
  a.layer = d->layer != 0, a.branch_norm = d->branch_norm != 0, a.gate_token = d->gate_token != 0;
  a.param_bf16 = d->param_dtype == KF_DTYPE_BF16;
  return a;
}

}  // namespace
}  // namespace kf

extern "C" int kf_residual_norm_fwd(const void* x, const void* branch, const void* gate, const void* w, const void* s,
                                    const void* bw, const void* bs, void* y, void* h, float* stats, int64_t rows,
                                    const kf_residual_norm_desc* d, void* stream) {
  using namespace kf;
  clear_error();
  if (int rc = check_common("kf_residual_norm_fwd", d, x, w, rows)) return rc;
  KF_CHECK_ARG(h != nullptr && (branch == nullptr || y != nullptr), "kf_residual_norm_fwd: null output");
  KF_CHECK_ARG(branch != nullptr || (gate == nullptr && !d->branch_norm && d->residual_scale == 1.f),
               "kf_residual_norm_fwd: a gate, a branch norm or a residual scale needs a branch");
  KF_CHECK_ARG(!d->branch_norm || bw != nullptr, "kf_residual_norm_fwd: the branch norm has no weight");
  if (rows == 0) return KF_OK;
  if (int rc = bind_device(x)) return rc;
  RowArgs a = row_args(d, rows);
  a.x = x, a.branch = branch, a.gate = gate, a.w = w, a.s = s, a.bw = bw, a.bs = bs, a.y = y, a.h = h;
  a.stats = reinterpret_cast<float4*>(stats);
  const bool vec = rows_aligned({x, branch, gate, w, s, bw, bs, y, h}, d->width);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  using bf = __nv_bfloat16;
  if (d->x_dtype == KF_DTYPE_BF16) return vec ? dispatch_fwd<true, bf, bf>(a, st) : dispatch_fwd<false, bf, bf>(a, st);
  if (d->branch_dtype == KF_DTYPE_BF16)
    return vec ? dispatch_fwd<true, float, bf>(a, st) : dispatch_fwd<false, float, bf>(a, st);
  return vec ? dispatch_fwd<true, float, float>(a, st) : dispatch_fwd<false, float, float>(a, st);
}

extern "C" int64_t kf_residual_norm_workspace(int64_t rows, int32_t width) {
  if (rows < 0 || width < 1 || width > kf::kMaxWidth) return 0;
  return (int64_t)kf::bwd_ctas(rows) * kf::kParamGrads * width;
}

extern "C" int kf_residual_norm_bwd(const void* x, const void* branch, const void* gate, const void* w, const void* bw,
                                    const void* bs, const float* stats, const void* dy, const void* dh,
                                    void* dx, void* dbranch, void* dgate, void* dw, void* ds, void* dbw, void* dbs,
                                    float* workspace, int64_t rows, const kf_residual_norm_desc* d, void* stream) {
  using namespace kf;
  clear_error();
  if (int rc = check_common("kf_residual_norm_bwd", d, x, w, rows)) return rc;
  KF_CHECK_ARG(workspace != nullptr && (rows == 0 || (stats != nullptr && dx != nullptr)), "kf_residual_norm_bwd: null argument");
  KF_CHECK_ARG(rows == 0 || branch == nullptr || dbranch != nullptr, "kf_residual_norm_bwd: the branch needs dbranch");
  KF_CHECK_ARG(rows == 0 || gate == nullptr || !d->gate_token || dgate != nullptr, "kf_residual_norm_bwd: the token gate needs dgate");
  KF_CHECK_ARG(!d->branch_norm || bw != nullptr, "kf_residual_norm_bwd: the branch norm has no weight");
  if (int rc = bind_device(workspace)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int ctas = 0;
  if (rows > 0) {
    GradArgs p{};
    p.f = row_args(d, rows);
    p.f.x = x, p.f.branch = branch, p.f.gate = gate, p.f.w = w, p.f.bw = bw, p.f.bs = bs;
    p.f.stats = const_cast<float4*>(reinterpret_cast<const float4*>(stats));
    p.dy = dy, p.dh = dh, p.dx = dx, p.dbranch = dbranch, p.dgate = dgate, p.part = workspace;
    ctas = bwd_ctas(rows);
    const bool vec = rows_aligned({x, branch, gate, w, bw, bs, dy, dh, dx, dbranch, d->gate_token ? dgate : nullptr}, d->width);
    using bf = __nv_bfloat16;
    int rc;
    if (d->x_dtype == KF_DTYPE_BF16)
      rc = vec ? dispatch_bwd<true, bf, bf>(p, ctas, st) : dispatch_bwd<false, bf, bf>(p, ctas, st);
    else if (d->branch_dtype == KF_DTYPE_BF16)
      rc = vec ? dispatch_bwd<true, float, bf>(p, ctas, st) : dispatch_bwd<false, float, bf>(p, ctas, st);
    else
      rc = vec ? dispatch_bwd<true, float, float>(p, ctas, st) : dispatch_bwd<false, float, float>(p, ctas, st);
    if (rc) return rc;
  }
  ParamOut o{{dw, ds, d->gate_token ? nullptr : dgate, dbw, dbs}};
  residual_norm_params<<<dim3((unsigned)cdiv(d->width, 32), kParamGrads), 256, 0, st>>>(workspace, ctas, d->width, o,
                                                                                        d->param_dtype == KF_DTYPE_BF16);
  return check_launch("kf_residual_norm_bwd");
}
