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
// shuffles and warps by one exchange in shared memory.  Those dependent steps leave
// memory idle, so each group of warps keeps its next rows coming by bulk copies
// into a ring of its own.  Everything between the loads and the stores is float32.
//
// Measured, cold caches: 32768 rows of 768 bf16, both norms, a gate per channel:
// forward 67 us (3.0 TB/s; 135 us without the rings), backward 113 us (2.7 TB/s) and
// 7 us for the parameters; 8192 rows of 4096 float32, a gate per token: forward 132 us
// (5.1 TB/s), backward 247 us (4.3 TB/s).  The measured copy rate is 6.6 TB/s.
// The bf16 forward issues in 70% of its slots; the backward falls short by what a row
// costs between its exchanges: the column sums take registers that more rows in
// flight would need.
#include <type_traits>

#include "f32x2.cuh"
#include "umma.cuh"

namespace kf {
namespace {

constexpr int kMaxWidth = 8192;
// Column sums of the backward.  With A = g (a gate per channel, or none) or
// A = gate g (a gate per token), every parameter gradient follows from four:
//   sum dh yhat = dw, sum dh = ds, sum A bhat, sum A,
// since dw_b = gate sum A bhat, ds_b = gate sum A and dgate = w_b sum A bhat + s_b sum A
// for a gate per channel.
constexpr int kSums = 4;

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
  float* part;  // (gridDim.x, kSums, width)
};

// Elements of a row owned by a lane, in V chunks of 8.  Aligned rows (width a
// multiple of 8) are read in 16-byte vectors; other rows element by element,
// lanes on neighbouring elements.
template <bool VEC>
__device__ __forceinline__ int elem(int c, int k, int warps, int wl) {
  return VEC ? (c * warps * 32 + wl) * 8 + k : (c * 8 + k) * warps * 32 + wl;
}

// A chunk is four pairs of float32.  Elements past the width are 0.
using Chunk = uint64_t[4];

__device__ __forceinline__ void load8(const float* p, Chunk& v) {
  const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(p), b = *reinterpret_cast<const ulonglong2*>(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, Chunk& v) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
__device__ __forceinline__ void store8(float* p, const Chunk& v) {
  *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(v[0], v[1]);
  *reinterpret_cast<ulonglong2*>(p + 4) = make_ulonglong2(v[2], v[3]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const Chunk& v) {
  uint4 a;
  uint32_t* w = &a.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    unpair(v[i], lo, hi);
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  *reinterpret_cast<uint4*>(p) = a;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_chunk(const T* row, int width, int c, int warps, int wl, Chunk& v) {
  if (VEC) {
    const int e = elem<true>(c, 0, warps, wl);
    if (e < width) {
      load8(row + e, v);
    } else {
      v[0] = v[1] = v[2] = v[3] = 0;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int e0 = elem<false>(c, 2 * k, warps, wl), e1 = elem<false>(c, 2 * k + 1, warps, wl);
      v[k] = pair(e0 < width ? to_f32<T>(row[e0]) : 0.f, e1 < width ? to_f32<T>(row[e1]) : 0.f);
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_chunk(T* row, int width, int c, int warps, int wl, const Chunk& v) {
  if (VEC) {
    const int e = elem<true>(c, 0, warps, wl);
    if (e < width) store8(row + e, v);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float lo, hi;
      unpair(v[k], lo, hi);
      const int e0 = elem<false>(c, 2 * k, warps, wl), e1 = elem<false>(c, 2 * k + 1, warps, wl);
      if (e0 < width) row[e0] = from_f32<T>(lo);
      if (e1 < width) row[e1] = from_f32<T>(hi);
    }
  }
}

// Parameters do not change while the kernel runs: read-only loads, which may
// go out ahead of the stores before them.
template <bool VEC>
__device__ __forceinline__ void load_param(const void* p, bool bf16, int width, int c, int warps, int wl, Chunk& v) {
  if (VEC) {
    const int e = elem<true>(c, 0, warps, wl);
    v[0] = v[1] = v[2] = v[3] = 0;
    if (e >= width) return;
    if (bf16) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + e));
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
      const float4 *f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + e), a = __ldg(f), b = __ldg(f + 1);
      v[0] = pair(a.x, a.y), v[1] = pair(a.z, a.w), v[2] = pair(b.x, b.y), v[3] = pair(b.z, b.w);
    }
    return;
  }
  if (bf16)
    load_chunk<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16*>(p), width, c, warps, wl, v);
  else
    load_chunk<float, VEC>(static_cast<const float*>(p), width, c, warps, wl, v);
}

// The parameters of the backward by column, with what stands for those not given.
enum { kW, kBranchW, kBranchS, kGate, kParams };

__device__ __forceinline__ float param_at(const void* p, bool bf16, int i) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ float param_of(const RowArgs& a, int which, int i) {
  const void* p = which == kW ? a.w : which == kGate ? (a.gate_token ? nullptr : a.gate) : !a.branch_norm ? nullptr : which == kBranchW ? a.bw : a.bs;
  return p != nullptr ? param_at(p, a.param_bf16, i) : which == kBranchS ? 0.f : 1.f;
}

// One of them for a chunk: from the float32 copy in shared memory, or from memory.
template <bool COPY, bool VEC>
__device__ __forceinline__ void get_param(const RowArgs& a, const float* copy, int which, int c, int wl, Chunk& v) {
  if (COPY) {
    load_chunk<float, VEC>(copy + which * a.width, a.width, c, a.warps, wl, v);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e0 = elem<VEC>(c, 2 * k, a.warps, wl), e1 = elem<VEC>(c, 2 * k + 1, a.warps, wl);
    v[k] = pair(e0 < a.width ? param_of(a, which, e0) : 0.f, e1 < a.width ? param_of(a, which, e1) : 0.f);
  }
}

// (v - mean) rstd w + s of one chunk; past the width w and s are 0, and so is it.
template <bool VEC>
__device__ __forceinline__ void affine(const RowArgs& a, const void* weight, const void* shift, float mean, float rstd, int c, int wl,
                                       const Chunk& v, Chunk& out) {
  Chunk w, s;
  load_param<VEC>(weight, a.param_bf16, a.width, c, a.warps, wl, w);
  if (shift != nullptr)
    load_param<VEC>(shift, a.param_bf16, a.width, c, a.warps, wl, s);
  else
    s[0] = s[1] = s[2] = s[3] = 0;
  const uint64_t r2 = pair(rstd), minus = pair(-mean);
#pragma unroll
  for (int k = 0; k < 4; ++k) out[k] = fma2(add2(v[k], minus), mul2(r2, w[k]), s[k]);
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

  // Both sums for the price of one: the lower half of the lanes goes on with a, the upper with b.
  __device__ __forceinline__ void sum2(float& a, float& b) {
    const bool low = lane < 16;
    float v = (low ? a : b) + __shfl_xor_sync(0xffffffffu, low ? b : a, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (warps == 1) {
      a = __shfl_sync(0xffffffffu, v, 0), b = __shfl_sync(0xffffffffu, v, 16);
      return;
    }
    float* p = buf + phase * warps * 3;
    phase ^= 1;
    if ((lane & 15) == 0) p[warp * 2 + (lane >> 4)] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
    a = b = 0.f;
    for (int w = 0; w < warps; ++w) a += p[w * 2], b += p[w * 2 + 1];
  }

  // Mean and reciprocal standard deviation of the group's row.  "layer": the
  // squares are taken about the warp's own mean and the warps' moments merged,
  // so a large mean costs no digits and one exchange is enough.
  template <int V, bool VEC>
  __device__ __forceinline__ float2 moments(const Chunk (&v)[V], int width, int wl, float eps, bool layer) {
    uint64_t acc = 0;
    if (!layer) {
#pragma unroll
      for (int c = 0; c < V; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc = fma2(v[c][k], v[c][k], acc);  // elements past the width are 0
      float sq = sum_of(acc), none = 0.f;
      sum2(sq, none);
      return make_float2(0.f, 1.f / sqrtf(sq / width + eps));
    }
#pragma unroll
    for (int c = 0; c < V; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc = add2(acc, v[c][k]);
    const float sum = warp_sum(sum_of(acc));
    float n = width, mean = sum / width;
    if (warps > 1) {
      n = 0.f;
#pragma unroll
      for (int c = 0; c < V; ++c)
        if (VEC) {
          n += elem<true>(c, 0, warps, wl) < width ? 8.f : 0.f;
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) n += elem<false>(c, k, warps, wl) < width ? 1.f : 0.f;
        }
      n = warp_sum(n);
      mean = n > 0.f ? sum / n : 0.f;
    }
    acc = 0;
    const uint64_t minus = pair(-mean);
#pragma unroll
    for (int c = 0; c < V; ++c) {
      if (VEC && elem<true>(c, 0, warps, wl) >= width) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint64_t d = add2(v[c][k], minus);
        if (!VEC) {
          float lo, hi;
          unpair(d, lo, hi);
          d = pair(elem<false>(c, 2 * k, warps, wl) < width ? lo : 0.f, elem<false>(c, 2 * k + 1, warps, wl) < width ? hi : 0.f);
        }
        acc = fma2(d, d, acc);
      }
    }
    float sq = sum_of(acc);
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

constexpr int kMaxTensors = 5;

// The rows a group of warps reads, some ahead: the slots are taken in turn and
// hold one row, one tensor after another.  Lane 0 of the group starts the copies;
// a slot is refilled once every lane has passed a barrier after its row.
struct RowRing {
  const uint8_t* from[kMaxTensors];  // the next row to start, of each tensor
  uint32_t bytes[kMaxTensors];       // of a row; 0: no such tensor
  uint8_t* data;
  uint64_t* full;
  int64_t rows, next, step;  // next: the row that from points to
  int slots, slot_bytes, put, get;
  uint32_t phase;
  bool leader, gave_up;

  __device__ __forceinline__ void init(uint8_t* at, uint64_t* barriers, int slots_, int slot_bytes_, int64_t rows_, int64_t first,
                                       int64_t step_, bool leader_) {
    data = at, full = barriers, slots = slots_, slot_bytes = slot_bytes_, rows = rows_, next = first, step = step_;
    leader = leader_, gave_up = false, put = get = 0, phase = 0;
  }
  __device__ __forceinline__ void tensor(int t, const void* p, uint32_t row_bytes) {
    bytes[t] = row_bytes;
    from[t] = static_cast<const uint8_t*>(p) + next * row_bytes;
  }
  __device__ __forceinline__ void start() {  // one more row, if there is one
    if (!leader || next >= rows) return;
    uint32_t total = 0;
#pragma unroll
    for (int t = 0; t < kMaxTensors; ++t) total += bytes[t];
    umma::mbar_arrive_expect_tx(full + put, total);
    uint8_t* to = data + put * slot_bytes;
#pragma unroll
    for (int t = 0; t < kMaxTensors; ++t) {
      if (bytes[t] == 0) continue;
      umma::bulk_load(to, from[t], bytes[t], full + put);
      from[t] += step * bytes[t];
      to += bytes[t];
    }
    next += step;
    if (++put == slots) put = 0;
  }
  // The next row.  A wait that ran out is recorded; the group goes on, so that no warp is left at a barrier.
  __device__ __forceinline__ const uint8_t* wait() {
    int abort = 0;
    if (!gave_up) gave_up = !umma::mbar_wait(full + get, phase, &abort);
    const uint8_t* at = data + get * slot_bytes;
    if (++get == slots) get = 0, phase ^= 1;
    return at;
  }
};

constexpr int kMaxSlots = 4;
constexpr int kFwdWarps = 16, kFwdRingWarps = 12;  // of a CTA of the forward, at most

template <int V, bool VEC, bool RING, typename TX, typename TB>
__global__ void __launch_bounds__((RING ? kFwdRingWarps : kFwdWarps) * 32, RING && sizeof(TX) == 2 ? 2 : 1) residual_norm_fwd(const RowArgs a, int slots, int slot_bytes) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint64_t full[8 * kMaxSlots];
  const int lane = threadIdx.x & 31, warp_id = threadIdx.x >> 5, group = warp_id / a.warps;
  const int groups = blockDim.x / 32 / a.warps;
  float* exch = reinterpret_cast<float*>(smem + (RING ? (size_t)groups * slots * slot_bytes : 0));
  RowGroup g{exch + group * 2 * a.warps * 3, a.warps, warp_id - group * a.warps, lane, 1 + group, 0};
  const int wl = g.warp * 32 + lane;
  const int64_t first = (int64_t)blockIdx.x * groups + group, step = (int64_t)gridDim.x * groups;
  RowRing ring;
  const uint32_t bx = a.width * sizeof(TX), bb = a.width * sizeof(TB);
  if (RING) {
    ring.init(smem + (size_t)group * slots * slot_bytes, full + group * kMaxSlots, slots, slot_bytes, a.rows, first, step, wl == 0);
    ring.tensor(0, a.x, bx);
    ring.tensor(1, a.branch, a.branch != nullptr ? bb : 0);
    ring.tensor(2, a.gate, a.gate_token ? bb : 0);
    ring.tensor(3, nullptr, 0), ring.tensor(4, nullptr, 0);
    if (threadIdx.x == 0) {
      for (int i = 0; i < groups * kMaxSlots; ++i) umma::mbar_init(full + i, 1);
      umma::fence_barrier_init();
    }
    __syncthreads();
    for (int i = 0; i < slots; ++i) ring.start();
  }
  for (int64_t row = first; row < a.rows; row += step) {
    const uint8_t* slot = RING ? ring.wait() : nullptr;
    const TX* xr = RING ? reinterpret_cast<const TX*>(slot) : static_cast<const TX*>(a.x) + row * a.width;
    const TB* br = RING ? reinterpret_cast<const TB*>(slot + bx) : static_cast<const TB*>(a.branch) + row * a.width;
    const TB* gr = RING ? reinterpret_cast<const TB*>(slot + bx + bb) : static_cast<const TB*>(a.gate) + row * a.width;
    Chunk y[V];
    float2 sb = make_float2(0.f, 1.f);
    if (a.branch != nullptr) {
      Chunk u[V];
#pragma unroll
      for (int c = 0; c < V; ++c) load_chunk<TB, VEC>(br, a.width, c, a.warps, wl, u[c]);
      if (!RING) {  // both loads under way before the first is waited for
#pragma unroll
        for (int c = 0; c < V; ++c) load_chunk<TX, VEC>(xr, a.width, c, a.warps, wl, y[c]);
      }
      if (a.branch_norm) {
        sb = g.moments<V, VEC>(u, a.width, wl, a.eps, a.layer);
#pragma unroll
        for (int c = 0; c < V; ++c) affine<VEC>(a, a.bw, a.bs, sb.x, sb.y, c, wl, u[c], u[c]);
      }
      const uint64_t alpha = pair(a.alpha);
#pragma unroll
      for (int c = 0; c < V; ++c) {
        if (RING) load_chunk<TX, VEC>(xr, a.width, c, a.warps, wl, y[c]);
        Chunk t = {pair(1.f), pair(1.f), pair(1.f), pair(1.f)};
        if (a.gate_token)
          load_chunk<TB, VEC>(gr, a.width, c, a.warps, wl, t);
        else if (a.gate != nullptr)
          load_param<VEC>(a.gate, a.param_bf16, a.width, c, a.warps, wl, t);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[c][k] = fma2(u[c][k], t[k], mul2(alpha, y[c][k]));
        store_chunk<TX, VEC>(static_cast<TX*>(a.y) + row * a.width, a.width, c, a.warps, wl, y[c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < V; ++c) load_chunk<TX, VEC>(xr, a.width, c, a.warps, wl, y[c]);
    }
    const float2 sy = g.moments<V, VEC>(y, a.width, wl, a.eps, a.layer);
    if (RING) {
      __syncwarp();  // with several warps the exchange in moments() was the barrier
      ring.start();
    }
#pragma unroll
    for (int c = 0; c < V; ++c) {
      affine<VEC>(a, a.w, a.s, sy.x, sy.y, c, wl, y[c], y[c]);
      store_chunk<TB, VEC>(static_cast<TB*>(a.h) + row * a.width, a.width, c, a.warps, wl, y[c]);
    }
    if (a.stats != nullptr && wl == 0) a.stats[row] = make_float4(sy.x, sy.y, sb.x, sb.y);
  }
}

// One CTA walks over rows blockIdx.x * groups + group, + gridDim.x * groups, ...
// The column sums stay with the lane that owns the columns, in registers for
// widths to 4096, in shared memory above, and become one partial
// sum per CTA in `part`.
template <int V, bool REGS, bool VEC, typename TX, typename TB>
__global__ void __launch_bounds__(REGS && V > 1 ? 256 : 512) residual_norm_bwd(const GradArgs p, int slots, int slot_bytes) {
  constexpr bool RING = VEC && REGS;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint64_t full[16 * kMaxSlots];
  const RowArgs& a = p.f;
  const int lane = threadIdx.x & 31, warp_id = threadIdx.x >> 5, group = warp_id / a.warps;
  const int groups = blockDim.x / 32 / a.warps;
  float* sums = reinterpret_cast<float*>(smem);  // (kSums, width); with the sums in registers the rings lie here until the end
  float* params = reinterpret_cast<float*>(smem + max((size_t)groups * slots * slot_bytes, sizeof(float) * kSums * a.width));
  float* exch = params + (REGS ? kParams * a.width : 0);
  RowGroup g{exch + group * 2 * a.warps * 3, a.warps, warp_id - group * a.warps, lane, 1 + group, 0};
  const int wl = g.warp * 32 + lane;
  Chunk acc[REGS ? kSums : 1][V] = {};
  const int64_t first = (int64_t)blockIdx.x * groups + group, step = (int64_t)gridDim.x * groups;
  RowRing ring;
  const uint32_t bx = a.width * sizeof(TX), bb = a.width * sizeof(TB);
  const bool branch = a.branch != nullptr, has_dy = p.dy != nullptr, has_dh = p.dh != nullptr;
  if (RING) {
    ring.init(smem + (size_t)group * slots * slot_bytes, full + group * kMaxSlots, slots, slot_bytes, a.rows, first, step, wl == 0);
    ring.tensor(0, a.x, bx);
    ring.tensor(1, p.dy, has_dy ? bx : 0);
    ring.tensor(2, p.dh, has_dh ? bb : 0);
    ring.tensor(3, a.branch, branch ? bb : 0);
    ring.tensor(4, a.gate, a.gate_token ? bb : 0);
    if (threadIdx.x == 0) {
      for (int i = 0; i < groups * kMaxSlots; ++i) umma::mbar_init(full + i, 1);
      umma::fence_barrier_init();
    }
    __syncthreads();
    for (int i = 0; i < slots; ++i) ring.start();
  } else {
    for (int i = threadIdx.x; i < kSums * a.width; i += blockDim.x) sums[i] = 0.f;
  }
  if (REGS)
    for (int i = threadIdx.x; i < a.width; i += blockDim.x)
#pragma unroll
      for (int j = 0; j < kParams; ++j) params[j * a.width + i] = param_of(a, j, i);
  __syncthreads();
  const float inv = 1.f / a.width;

  // sums j of chunk c, pair k
  auto add = [&](int j, int c, int k, uint64_t v, uint64_t w) {  // += v w
    if (REGS) {
      acc[REGS ? j : 0][c][k] = fma2(v, w, acc[REGS ? j : 0][c][k]);
    } else {
      float lo, hi;
      unpair(mul2(v, w), lo, hi);
      const int e0 = elem<VEC>(c, 2 * k, a.warps, wl), e1 = elem<VEC>(c, 2 * k + 1, a.warps, wl);
      if (e0 < a.width) sums[j * a.width + e0] += lo;
      if (e1 < a.width) sums[j * a.width + e1] += hi;
    }
  };
  const uint64_t one = pair(1.f), alpha = pair(a.alpha);
  for (int64_t row = first; row < a.rows; row += step) {
    const int64_t off = row * a.width;
    const float4 st = a.stats[row];
    const uint8_t* slot = RING ? ring.wait() : nullptr;
    // this row of each tensor, in the ring or in global memory
    const uint8_t *s_dy = slot + bx, *s_dh = s_dy + (has_dy ? bx : 0), *s_br = s_dh + (has_dh ? bb : 0), *s_gate = s_br + (branch ? bb : 0);
    const TX* xr = RING ? reinterpret_cast<const TX*>(slot) : static_cast<const TX*>(a.x) + off;
    const TX* dyr = RING ? reinterpret_cast<const TX*>(s_dy) : static_cast<const TX*>(p.dy) + off;
    const TB* dhr = RING ? reinterpret_cast<const TB*>(s_dh) : static_cast<const TB*>(p.dh) + off;
    const TB* brr = RING ? reinterpret_cast<const TB*>(s_br) : static_cast<const TB*>(a.branch) + off;
    const TB* gater = RING ? reinterpret_cast<const TB*>(s_gate) : static_cast<const TB*>(a.gate) + off;
    const float2 bst = a.branch_norm ? make_float2(st.z, st.w) : make_float2(0.f, 1.f);
    Chunk hat[V], dh[V], gr[V], bhat[V];
    uint64_t s1 = 0, s2 = 0;
    // y again, from x and the branch and not from its rounded copy: as many bytes to read, and no rounding in yhat
#pragma unroll
    for (int c = 0; c < V; ++c) {
      load_chunk<TX, VEC>(xr, a.width, c, a.warps, wl, hat[c]);
      if (has_dh)
        load_chunk<TB, VEC>(dhr, a.width, c, a.warps, wl, dh[c]);
      else
        dh[c][0] = dh[c][1] = dh[c][2] = dh[c][3] = 0;
      if (branch) {
        Chunk w, t, f;
        load_chunk<TB, VEC>(brr, a.width, c, a.warps, wl, bhat[c]);
        get_param<REGS, VEC>(a, params, kBranchW, c, wl, w);
        get_param<REGS, VEC>(a, params, kBranchS, c, wl, t);
        if (a.gate_token)
          load_chunk<TB, VEC>(gater, a.width, c, a.warps, wl, f);
        else
          get_param<REGS, VEC>(a, params, kGate, c, wl, f);
        const uint64_t rstd = pair(bst.y), minus = pair(-bst.x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          bhat[c][k] = mul2(add2(bhat[c][k], minus), rstd);
          hat[c][k] = fma2(fma2(bhat[c][k], w[k], t[k]), f[k], mul2(alpha, hat[c][k]));
        }
      }
      Chunk w;
      get_param<REGS, VEC>(a, params, kW, c, wl, w);
      const uint64_t rstd = pair(st.y), minus = pair(-st.x);
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // past the width dh is 0, and no sum is kept
        hat[c][k] = mul2(add2(hat[c][k], minus), rstd);
        add(0, c, k, dh[c][k], hat[c][k]);
        add(1, c, k, dh[c][k], one);
        dh[c][k] = mul2(dh[c][k], w[k]);
        s1 = add2(s1, dh[c][k]);
        s2 = fma2(dh[c][k], hat[c][k], s2);
      }
    }
    float m1 = sum_of(s1), m2 = sum_of(s2);
    g.sum2(m1, m2);
    if (RING && !a.branch_norm && row != first) ring.start();  // every lane is done with the row before
    m1 = a.layer ? m1 * inv : 0.f;
    m2 *= inv;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      if (has_dy)
        load_chunk<TX, VEC>(dyr, a.width, c, a.warps, wl, gr[c]);
      else
        gr[c][0] = gr[c][1] = gr[c][2] = gr[c][3] = 0;
      const uint64_t rstd = pair(st.y), a1 = pair(-m1), a2 = pair(-m2);
      Chunk t;
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // dy + rstd (dh - m1 - yhat m2)
        gr[c][k] = fma2(fma2(hat[c][k], a2, add2(dh[c][k], a1)), rstd, gr[c][k]);
        t[k] = mul2(alpha, gr[c][k]);
      }
      store_chunk<TX, VEC>(static_cast<TX*>(p.dx) + off, a.width, c, a.warps, wl, t);
    }
    if (!branch) continue;
    // from here dh holds du w_b
    s1 = s2 = 0;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      Chunk w, t;
      get_param<REGS, VEC>(a, params, kBranchW, c, wl, w);
      if (a.gate_token) {
        Chunk u;
        get_param<REGS, VEC>(a, params, kBranchS, c, wl, u);
        load_chunk<TB, VEC>(gater, a.width, c, a.warps, wl, t);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          u[k] = mul2(fma2(bhat[c][k], w[k], u[k]), gr[c][k]);
          gr[c][k] = mul2(gr[c][k], t[k]);
        }
        store_chunk<TB, VEC>(static_cast<TB*>(p.dgate) + off, a.width, c, a.warps, wl, u);
      }
      if (!a.gate_token) get_param<REGS, VEC>(a, params, kGate, c, wl, t);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        add(2, c, k, gr[c][k], bhat[c][k]);
        add(3, c, k, gr[c][k], one);
        if (!a.gate_token) gr[c][k] = mul2(gr[c][k], t[k]);
      }
      if (a.branch_norm) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          dh[c][k] = mul2(gr[c][k], w[k]);
          s1 = add2(s1, dh[c][k]);
          s2 = fma2(dh[c][k], bhat[c][k], s2);
        }
      } else {
        store_chunk<TB, VEC>(static_cast<TB*>(p.dbranch) + off, a.width, c, a.warps, wl, gr[c]);
      }
    }
    if (!a.branch_norm) continue;
    m1 = sum_of(s1), m2 = sum_of(s2);
    g.sum2(m1, m2);
    if (RING) ring.start();  // these sums took all that the row's slot holds
    const uint64_t rstd = pair(st.w), a1 = pair(a.layer ? -m1 * inv : 0.f), a2 = pair(-m2 * inv);
#pragma unroll
    for (int c = 0; c < V; ++c) {
#pragma unroll
      for (int k = 0; k < 4; ++k) dh[c][k] = mul2(fma2(bhat[c][k], a2, add2(dh[c][k], a1)), rstd);
      store_chunk<TB, VEC>(static_cast<TB*>(p.dbranch) + off, a.width, c, a.warps, wl, dh[c]);
    }
  }

  // the groups' sums join in group order
  if (REGS) {
    if (RING) {
      __syncthreads();
      for (int i = threadIdx.x; i < kSums * a.width; i += blockDim.x) sums[i] = 0.f;
    }
    for (int r = 0; r < groups; ++r) {
      __syncthreads();
      if (r == group) {
#pragma unroll
        for (int j = 0; j < kSums; ++j)
#pragma unroll
          for (int c = 0; c < V; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float lo, hi;
              unpair(acc[REGS ? j : 0][c][k], lo, hi);
              const int e0 = elem<VEC>(c, 2 * k, a.warps, wl), e1 = elem<VEC>(c, 2 * k + 1, a.warps, wl);
              if (e0 < a.width) sums[j * a.width + e0] += lo;
              if (e1 < a.width) sums[j * a.width + e1] += hi;
            }
      }
    }
  }
  __syncthreads();
  float* out = p.part + (int64_t)blockIdx.x * kSums * a.width;
  for (int i = threadIdx.x; i < kSums * a.width; i += blockDim.x) out[i] = sums[i];
}

struct ParamOut {
  void *dw, *ds, *dgate, *dbw, *dbs;  // null: not wanted
};

// Column sums of the CTAs' partial sums, in a fixed order: 32 columns by 16
// slices of the CTAs, slices joined in order.
__global__ void __launch_bounds__(512) residual_norm_params(const float* part, int n_part, const RowArgs a, ParamOut o) {
  __shared__ float s[kSums][16][33];
  const int lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane, slice = threadIdx.x >> 5;
  float v[kSums] = {};
  if (col < a.width) {
#pragma unroll 4
    for (int i = slice; i < n_part; i += 16)
#pragma unroll
      for (int j = 0; j < kSums; ++j) v[j] += part[((int64_t)i * kSums + j) * a.width + col];
  }
#pragma unroll
  for (int j = 0; j < kSums; ++j) s[j][slice][lane] = v[j];
  __syncthreads();
  if (slice != 0 || col >= a.width) return;
#pragma unroll
  for (int j = 0; j < kSums; ++j)
    for (int i = 1; i < 16; ++i) v[j] += s[j][i][lane];
  auto put = [&](void* p, float x) {
    if (p == nullptr) return;
    if (a.param_bf16)
      static_cast<__nv_bfloat16*>(p)[col] = __float2bfloat16_rn(x);
    else
      static_cast<float*>(p)[col] = x;
  };
  put(o.dw, v[0]);
  put(o.ds, v[1]);
  const bool channel = a.gate != nullptr && !a.gate_token;
  const float gate = channel ? param_at(a.gate, a.param_bf16, col) : 1.f;
  if (channel) {
    float x = v[2];
    if (a.branch_norm) x = x * param_at(a.bw, a.param_bf16, col) + (a.bs != nullptr ? v[3] * param_at(a.bs, a.param_bf16, col) : 0.f);
    put(o.dgate, x);
  }
  if (a.branch_norm) {
    put(o.dbw, gate * v[2]);
    put(o.dbs, gate * v[3]);
  }
}

bool rows_aligned(std::initializer_list<const void*> ps, int width) {
  if (width % 8) return false;
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}


// CTAs of the backward: one per SM, fewer when there are fewer rows than CTAs.
int bwd_ctas(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>(rows, 148)); }

int sm_count() {
  int dev = 0, n = 0;
  const bool ok = cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess;
  return ok ? n : 148;
}

template <int V, bool VEC, bool RING, typename TX, typename TB>
int launch_fwd(RowArgs a, cudaStream_t s) {
  const int groups = std::max(1, 8 / a.warps);
  KF_CHECK_ARG(groups * a.warps <= (RING ? kFwdRingWarps : kFwdWarps), "kf_residual_norm_fwd: %d warps to a row of %d elements", a.warps, a.width);
  const int slot_bytes = a.width * (int)(sizeof(TX) + (a.branch != nullptr ? sizeof(TB) : 0) + (a.gate_token ? sizeof(TB) : 0));
  int slots = 0;
  const int per_sm = sizeof(TX) == 2 ? 3 : 2;  // CTAs
  if (RING)
    for (slots = kMaxSlots; slots > 1 && slots * groups * slot_bytes > 200 * 1024 / per_sm;) --slots;
  const size_t smem = (size_t)groups * slots * slot_bytes + groups * 2 * a.warps * 3 * sizeof(float);
  auto* k = residual_norm_fwd<V, VEC, RING, TX, TB>;
  static SmemAllowed allowed;
  if (int rc = allow_smem(k, smem, allowed)) return rc;
  const int64_t ctas = cdiv(a.rows, groups);
  k<<<(unsigned)(RING ? std::min<int64_t>(ctas, per_sm * sm_count()) : ctas), groups * a.warps * 32, smem, s>>>(a, slots, slot_bytes);
  return check_launch("kf_residual_norm_fwd");
}

template <int V, bool REGS, bool VEC, typename TX, typename TB>
int launch_bwd(GradArgs p, int ctas, cudaStream_t s) {
  const RowArgs& a = p.f;
  constexpr size_t kLimit = 226 * 1024;  // of shared memory, beside the barriers
  int groups = REGS && V > 1 ? 8 : std::max(1, 15 / a.warps);  // one named barrier each
  const int slot_bytes = a.width * (int)(sizeof(TX) * (1 + (p.dy != nullptr)) +
                                         sizeof(TB) * ((p.dh != nullptr) + (a.branch != nullptr) + a.gate_token));
  // what is kept beside the rings: the parameters (widths to 4096) and the exchange buffers
  const size_t beside = (REGS ? sizeof(float) * kParams * a.width : 0) + groups * 2 * a.warps * 3 * sizeof(float);
  int slots = 0;
  if (VEC && REGS) {
    for (slots = kMaxSlots; slots > 2 && slots * groups * slot_bytes + beside > kLimit;) --slots;
    // float32 rows of 700 to 768 elements with a gate per token: two slots for each of 8 warps are too much
    while (groups > 1 && slots * groups * slot_bytes + beside > kLimit) --groups;
  }
  const size_t smem = std::max<size_t>((size_t)groups * slots * slot_bytes, sizeof(float) * kSums * a.width) + beside;
  auto* k = residual_norm_bwd<V, REGS, VEC, TX, TB>;
  static SmemAllowed allowed1;
  if (int rc = allow_smem(k, smem, allowed1)) return rc;
  k<<<ctas, groups * a.warps * 32, smem, s>>>(p, slots, slot_bytes);
  return check_launch("kf_residual_norm_bwd");
}

// A lane takes 8 V elements of a row.  With many rows (16 chunks of 256 elements an
// SM) a row goes to as few warps as possible (a warp alone needs no exchange) and rows
// come through the rings: 32768 x 768 bf16 in 65 us, 135 us one row a group.  With
// few it is spread over more warps, one row a group: 3 rows of 768 in 5 us, where a
// ring has nothing to run ahead of.
template <bool VEC, typename TX, typename TB>
int dispatch_fwd(RowArgs a, cudaStream_t s) {
  const int chunks = (int)cdiv(a.width, 256);
  if constexpr (VEC) {
    if (a.rows * chunks >= 148 * 16) {
      int v = 1, least = 1 << 30;
      for (int t = 4; t >= 1; --t)
        if (cdiv(chunks, t) <= kFwdRingWarps && cdiv(chunks, t) * t < least) least = (int)cdiv(chunks, t) * t, v = t;
      a.warps = (int)cdiv(chunks, v);
      if (v == 4) return launch_fwd<4, VEC, true, TX, TB>(a, s);
      if (v == 3) return launch_fwd<3, VEC, true, TX, TB>(a, s);
      if (v == 2) return launch_fwd<2, VEC, true, TX, TB>(a, s);
      return launch_fwd<1, VEC, true, TX, TB>(a, s);
    }
  }
  const int v = chunks > 16 ? 2 : 1;
  a.warps = (int)cdiv(chunks, v);
  return v == 2 ? launch_fwd<2, VEC, false, TX, TB>(a, s) : launch_fwd<1, VEC, false, TX, TB>(a, s);
}

// Up to 768 columns a warp has a row to itself: its column sums fill the
// registers of 8 warps an SM, but no row waits at a barrier (32768 x 768: 112 us,
// 126 us with three warps to a row).  Above 4096 the sums do not fit the registers
// and are kept in shared memory.
template <bool VEC, typename TX, typename TB>
int dispatch_bwd(GradArgs p, int ctas, cudaStream_t s) {
  const int chunks = (int)cdiv(p.f.width, 256);
  if constexpr (VEC) {
    p.f.warps = 1;
    if (chunks == 2) return launch_bwd<2, true, VEC, TX, TB>(p, ctas, s);
    if (chunks == 3) return launch_bwd<3, true, VEC, TX, TB>(p, ctas, s);
  }
  const bool regs = p.f.width <= 4096;
  p.f.warps = (int)cdiv(chunks, regs ? 1 : 2);
  return regs ? launch_bwd<1, true, VEC, TX, TB>(p, ctas, s) : launch_bwd<2, false, VEC, TX, TB>(p, ctas, s);
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
  KF_CHECK_ARG(!d->gate_token || gate != nullptr, "kf_residual_norm_fwd: a gate per token is missing");
  KF_CHECK_ARG(reinterpret_cast<uintptr_t>(stats) % 16 == 0, "kf_residual_norm_fwd: stats must start at a multiple of 16 bytes");
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
  return (int64_t)kf::bwd_ctas(rows) * kf::kSums * width;
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
  KF_CHECK_ARG(rows == 0 || !d->gate_token || gate != nullptr, "kf_residual_norm_bwd: a gate per token is missing");
  KF_CHECK_ARG(reinterpret_cast<uintptr_t>(stats) % 16 == 0, "kf_residual_norm_bwd: stats must start at a multiple of 16 bytes");
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
  RowArgs a = row_args(d, rows);
  a.gate = gate, a.bw = bw, a.bs = bs;
  residual_norm_params<<<(unsigned)cdiv(d->width, 32), 512, 0, st>>>(workspace, ctas, a,
                                                                    ParamOut{dw, ds, d->gate_token ? nullptr : dgate, dbw, dbs});
  return check_launch("kf_residual_norm_bwd");
}
