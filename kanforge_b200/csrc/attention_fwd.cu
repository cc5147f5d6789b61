// Attention forward over packed sequences for bf16, on the tensor cores.
//
// A CTA owns 256 rows of one sequence and key head as two MMA tiles of 128.
// Rows are (query, head) pairs: the heads that share a key head are neighbouring
// rows, so each K and V tile serves all of them.  Per tile of 128 keys:
//   S = Q K^T into tensor memory; a softmax thread owns one row (a TMEM lane),
//   reads its 128 scores, keeps the running maximum and sum in registers and
//   writes P = 2^(t - m) back to tensor memory as bf16; O += P V with P as the
//   A operand from there.
// P is rounded to bf16 for the tensor cores (2^-9 of each weight, summed with
// either sign); the sum that divides O is the float32 one.  The maximum in use
// moves only when a row's true one is more than 8 above it (2^8 times the sum
// in float32 and bf16 loses nothing), so O is rarely rescaled.
// While one tile's softmax runs, the tensor cores work for the other tile.
// Warps 0-7 softmax (one warpgroup a tile), 8-10 load, 11 issues the MMAs.
#include "attention_tc.cuh"

namespace kf {
namespace {

using namespace attn;

constexpr int kThreads = 384, kLoaders = 96;
constexpr float kLazy = 8.f;

template <int DP>
struct Fwd {
  static constexpr int kStages = DP == 64 ? 6 : 4;  // K and V tiles in flight
  static constexpr int kTile = tile_bytes<DP>();
  static constexpr int kSmem = 1024 + (2 + kStages) * kTile;  // + bias tables
  // tensor memory columns; with DP = 64 there is room for P beside S
  static constexpr uint32_t o(int t) { return 256 + t * DP; }
  static constexpr uint32_t p(int t) { return DP == 64 ? 384 + t * 64 : t * 128; }
};

struct Ctl {
  uint64_t q_full, fin, kv_full[8], kv_empty[8], s_full[2], p_ready[2], o_done[2];
  uint32_t tmem;
  int abort;
};

template <int DP>
__global__ void __launch_bounds__(kThreads, 1) attention_fwd_tc(const Args a) {
  using F = Fwd<DP>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Ctl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sbias = reinterpret_cast<float*>(smem + (2 + F::kStages) * F::kTile);
  volatile int* abort = &ctl.abort;

  const int2 tile = a.tiles[blockIdx.x];
  const Seq s = load_seq(a, tile.x);
  const int pack = a.pack, head0 = blockIdx.y * pack, kv_head = head0 / (a.heads / a.kv_heads);
  const int r0 = tile.y * 2 * kRows, off = s.lk - s.lq, total = s.lq * pack;
  // key tiles of each of the two row tiles
  int n_rows[2], n_kv[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    n_rows[t] = min(kRows, max(0, total - r0 - t * kRows));
    const int last = (r0 + t * kRows + n_rows[t] - 1) / pack;  // its last query
    const int keys = n_rows[t] == 0 ? 0 : a.causal ? min(s.lk, last + off + 1) : s.lk;
    n_kv[t] = max(0, (keys + kRows - 1) / kRows);
  }
  const int n_max = max(n_kv[0], n_kv[1]);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    ctl.abort = 0;
    mbar_init(&ctl.q_full, kLoaders);
    mbar_init(&ctl.fin, 1);
    for (int i = 0; i < F::kStages; ++i) mbar_init(&ctl.kv_full[i], kLoaders), mbar_init(&ctl.kv_empty[i], 1);
    for (int t = 0; t < 2; ++t) mbar_init(&ctl.s_full[t], 1), mbar_init(&ctl.p_ready[t], kRows), mbar_init(&ctl.o_done[t], 1);
    fence_barrier_init();
  }
  if (warp == 11) {
    tmem_alloc(&ctl.tmem, 512);
    tmem_relinquish();
  }
  if (a.table != nullptr) expand_bias_padded(a, head0, pack, sbias, threadIdx.x, kThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl.tmem, q_tile = smem_u32(smem), kv_tile = q_tile + 2 * F::kTile;

  // registers: 384 x 168 at launch = 256 x 208 + 128 x 88
  if (warp >= 8) reg_dec<88>();
  if (warp >= 8 && warp < 11) {
    // ---- loads: Q, then K and V tiles in turn through the ring
    const int tid = threadIdx.x - 256;
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q.p) + (int64_t)s.q0 * a.q.row + head0 * a.q.head;
    const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(a.k.p) + (int64_t)s.k0 * a.k.row + kv_head * a.k.head;
    const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v.p) + (int64_t)s.k0 * a.v.row + kv_head * a.v.head;
#pragma unroll
    for (int t = 0; t < 2; ++t)
      load_tile_async<DP, kLoaders>(q_tile + t * F::kTile, q, a.q.row, a.q.head, pack, r0 + t * kRows, n_rows[t], a.dim, tid);
    feed_ring<F::kStages>(2 * n_max, &ctl.q_full, ctl.kv_full, ctl.kv_empty, abort, [&](int it) {
      const bool is_v = it & 1;
      const int j = it >> 1;
      load_tile_async<DP, kLoaders>(kv_tile + it % F::kStages * F::kTile, is_v ? v : k, is_v ? a.v.row : a.k.row, 0, 1, j * kRows,
                                    min(kRows, s.lk - j * kRows), a.dim, tid);
    });
  } else if (warp == 11) {
    // ---- MMAs
    if (lane == 0 && n_max > 0) {
      const uint32_t idesc_s = idesc_bf16_f32(kRows, kRows, false, false), idesc_o = idesc_bf16_f32(kRows, DP, false, true);
      auto full = [&](int it) { return mbar_wait(&ctl.kv_full[it % F::kStages], (it / F::kStages) & 1, abort); };
      auto last_user = [&](int j) { return n_kv[1] > j ? 1 : 0; };
      auto scores = [&](int t, int j) {
        if (!full(2 * j)) return false;
        tc_fence_after();
        const uint32_t kt = kv_tile + (2 * j % F::kStages) * F::kTile;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) mma_ss(tmem + t * 128, desc_k(q_tile + t * F::kTile, i), desc_k(kt, i), idesc_s, i > 0);
        mma_commit(&ctl.s_full[t]);
        if (t == last_user(j)) mma_commit(&ctl.kv_empty[2 * j % F::kStages]);
        return true;
      };
      bool ok = mbar_wait(&ctl.q_full, 0, abort);
      for (int t = 0; t < 2; ++t)
        if (ok && n_kv[t] > 0) ok = scores(t, 0);
      for (int j = 0; j < n_max && ok; ++j) {
        for (int t = 0; t < 2 && ok; ++t) {
          if (j >= n_kv[t]) continue;
          const int it = 2 * j + 1;
          if (!(ok = mbar_wait(&ctl.p_ready[t], j & 1, abort) && full(it))) break;
          tc_fence_after();
          const uint32_t vt = kv_tile + (it % F::kStages) * F::kTile;
#pragma unroll
          for (int i = 0; i < 8; ++i) mma_ts(tmem + F::o(t), tmem + F::p(t) + i * 8, desc_mn(vt, i), idesc_o, j > 0 || i > 0);
          mma_commit(&ctl.o_done[t]);
          if (t == last_user(j)) mma_commit(&ctl.kv_empty[it % F::kStages]);
          if (j + 1 < n_kv[t]) {
            // DP = 128: the next scores take P's columns, so P V has to be done
            if (DP == 128 && !(ok = mbar_wait(&ctl.o_done[t], j & 1, abort))) break;
            ok = scores(t, j + 1);
          }
        }
      }
      mma_commit(&ctl.fin);
      mbar_drain(&ctl.fin, 0);
    }
  } else {
    reg_inc<208>();
    // ---- softmax: thread = row
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const int r = r0 + t * kRows + row, n = n_kv[t];
    const bool valid = row < n_rows[t];
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int tok = r / pack, pos = tok + off;
    const int limit = valid && a.causal ? min(s.lk, pos + 1) : s.lk;  // keys this row sees
    const float c2 = a.scale * kLog2e;
    const float* bias = sbias + (a.table != nullptr ? (r - tok * pack) * bias_floats(a.span) + a.span + kBiasPad : 0);
    float m = -CUDART_INF_F, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      if (!(ok = mbar_wait_warp(&ctl.s_full[t], j & 1, abort))) break;
      tc_fence_after();
      float x[128];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld32_issue(lanes + t * 128 + i * 32, x + i * 32);
      tmem_wait_ld(x);
      const int k0 = j * kRows;
      float mul = c2, add = 0.f;
      if (a.table != nullptr) {
        const int dist = pos - k0;  // to the tile's first key
        const bool far = dist - (kRows - 1) >= a.span || dist <= -a.span;
        if (__all_sync(0xffffffffu, far)) {
          add = dist > 0 ? bias[a.span] : bias[-a.span];
        } else {
          const float* b = bias + max(-a.span - kBiasPad + kRows - 1, min(dist, a.span + kBiasPad));
#pragma unroll
          for (int i = 0; i < 128; ++i) x[i] = fmaf(x[i], c2, b[-i]);
          mul = 1.f;
        }
      }
      if (__any_sync(0xffffffffu, limit - k0 < kRows)) {
        const int seen = limit - k0;
#pragma unroll
        for (int i = 0; i < 128; ++i) x[i] = i < seen ? x[i] : -CUDART_INF_F;
      }
      float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int i = 4; i < 128; ++i) top[i & 3] = fmaxf(top[i & 3], x[i]);
      const float high = fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), mul, add);
      if (__any_sync(0xffffffffu, high > m + kLazy)) {
        // some row's maximum moves: its sum and output follow (O is idle: S came after the last P V)
        const float m_new = fmaxf(m, high);
        const float fix = m == -CUDART_INF_F ? 0.f : ex2(m - m_new);
        m = m_new;
        l *= fix;
        if (j > 0) {
#pragma unroll
          for (int i = 0; i < DP / 32; ++i) {
            float o[32];
            tmem_ld32_issue(lanes + F::o(t) + i * 32, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] *= fix;
            tmem_st32(lanes + F::o(t) + i * 32, reinterpret_cast<uint32_t*>(o));
          }
        }
      }
      const float base = add - (m == -CUDART_INF_F ? 0.f : m);  // a row without a visible key yet: 2^-inf = 0
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t p[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float e0 = ex2(fmaf(x[h * 64 + 2 * i], mul, base)), e1 = ex2(fmaf(x[h * 64 + 2 * i + 1], mul, base));
          sum[0] += e0;
          sum[1] += e1;
          p[i] = pack_bf16x2(e0, e1);
        }
        tmem_st32(lanes + F::p(t) + h * 32, p);
      }
      l += sum[0] + sum[1];
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&ctl.p_ready[t]);
    }
    // ---- O / l, and the logarithm of the sum
    if (ok && n > 0) ok = mbar_wait_warp(&ctl.o_done[t], (n - 1) & 1, abort);
    if (ok) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t at = ((int64_t)(s.q0 + tok) * a.heads + head0 + (r - tok * pack)) * a.dim;
      if (valid && a.lse != nullptr)
        a.lse[(int64_t)(head0 + (r - tok * pack)) * a.tq + s.q0 + tok] = l == 0.f ? 0.f : m + log2f(l);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        float o[32];
        __syncwarp();
        if (n > 0) {
          tmem_ld32_issue(lanes + F::o(t) + i * 32, o);
          tmem_wait_ld(o);
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = n > 0 && l != 0.f ? o[c] * inv : 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (!valid || i * 32 + q * 8 >= a.dim) continue;
          uint4 w;
          uint32_t* u = &w.x;
#pragma unroll
          for (int c = 0; c < 4; ++c) u[c] = pack_bf16x2(o[q * 8 + 2 * c], o[q * 8 + 2 * c + 1]);
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.o) + at + i * 32 + q * 8) = w;
          if (a.o_rest != nullptr) {
            uint4 e;
            uint32_t* f = &e.x;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              f[c] = pack_bf16x2(o[q * 8 + 2 * c] - __uint_as_float(u[c] << 16),
                                 o[q * 8 + 2 * c + 1] - __uint_as_float(u[c] & 0xffff0000u));
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.o_rest) + at + i * 32 + q * 8) = e;
          }
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 11) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DP>
int launch(const Args& a, int n_tiles, cudaStream_t st) {
  const size_t smem = Fwd<DP>::kSmem + (a.table != nullptr ? a.pack * bias_floats(a.span) * sizeof(float) : 0);
  KF_CUDA_RET(cudaFuncSetAttribute(attention_fwd_tc<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  attention_fwd_tc<DP><<<dim3(n_tiles, a.heads / a.pack), kThreads, smem, st>>>(a);
  return check_launch("kf_attention_fwd");
}

}  // namespace

namespace attn {
int fwd_bf16(const Args& a, int n_tiles, cudaStream_t st) { return a.dim <= 64 ? launch<64>(a, n_tiles, st) : launch<128>(a, n_tiles, st); }
}  // namespace attn
}  // namespace kf
