// Attention forward over packed sequences for bf16, on the tensor cores.
//
// A CTA owns one (D <= 64) or two row tiles of 128 of one sequence and key head.
// Rows are (query, head) pairs: the heads that share a key head are neighbouring
// rows, so each K and V tile serves all of them.  Per 64 keys:
//   S = Q K^T into tensor memory; a softmax thread owns one row (a TMEM lane),
//   reads its 64 scores, keeps the running maximum and sum in registers and
//   writes P = 2^(t - m) back to tensor memory as bf16; O += P V with P as the
//   A operand from there.
// P is rounded to bf16 for the tensor cores (2^-9 of each weight, summed with
// either sign); the sum that divides O is the float32 one.  The maximum in use
// moves only when a row's true one is more than 8 above it (2^8 times the sum
// in float32 and bf16 loses nothing), so O is rarely rescaled.
// Two scores of 64 keys are in flight for each row tile: the chain S -> softmax
// -> P V -> next S of one runs under the softmax of the other.  An SM holds two
// row tiles, all that tensor memory has room for: with D = 128 as one CTA, which
// reads K and V once for both; with D <= 64, where the exponentials and not the
// loads bound the loop, as two CTAs, so that one starts and ends under the other.
// Warps: softmax (four a row tile), one that loads, and for each row tile one that
// issues Q K^T and one that issues P V: issuing blocks while the tensor cores
// are behind, and neither product should wait for the other's turn.
//
// Measured, cold caches, causal: 8191 tokens, 16 heads of 128 on 4 key heads 0.24 ms
// (1.15 PFLOP/s, 0.70 of the measured bf16 rate); 32 x 1024 tokens, 12 heads of 64
// with a bias 0.18 ms (290 TFLOP/s); 64 x 197 tokens both ways with a bias 67 us, where
// about half of a CTA's time is its loop, the rest its set-up, queries, bias table
// and output: code that runs once costs the fetching of its instructions, so it is
// kept in loops (77 us unrolled).  No pipe is full: what the time goes to is the way
// of one row tile through a thread (scores out of tensor memory, maximum, 64
// exponentials, weights back), which two row tiles an SM do not hide altogether.
// The tensor cores wait for the weights, with D = 64 most of the time, since a
// product there is half as long and the exponentials are as many.  Two threads to
// a row would halve that way; that has not been tried.
#include "attention_tc.cuh"

namespace kf {
namespace {

using namespace attn;

constexpr float kLazy = 8.f;
constexpr int kKeys = 64;  // of one set of scores

template <int DP>
struct Fwd {
  static constexpr int NT = DP == 64 ? 1 : 2;          // row tiles
  static constexpr int kUnit = DP == 64 ? 64 : 128;    // keys of a streamed tile
  static constexpr int kStages = DP == 64 ? 10 : 4;    // K and V tiles in flight
  static constexpr int kTile = tile_bytes<DP>(kUnit), kQTile = tile_bytes<DP>(kRows);
  static constexpr int kSmem = 1024 + NT * kQTile + kStages * kTile;  // + bias tables
  static constexpr int kSoftmax = NT * 128, kLoadWarp = NT * 4, kMmaWarp = DP == 64 ? 5 : 12;
  static constexpr int kThreads = DP == 64 ? 256 : 512;
  // registers: 128 a thread at launch, as many for the softmax and the other half of the warps together
  static constexpr int kSoftmaxRegs = DP == 64 ? 192 : 200, kOtherRegs = 256 - kSoftmaxRegs;
  static constexpr uint32_t kCols = DP == 64 ? 256 : 512;
  // tensor memory columns; with D <= 64 there is room for P beside S, with 128 it takes the columns of its scores
  __device__ static constexpr uint32_t s(int t, int h) { return t * 128 + h * kKeys; }
  __device__ static constexpr uint32_t o(int t) { return NT * 128 + t * DP; }
  __device__ static constexpr uint32_t p(int t, int h) { return DP == 64 ? 192 + h * 32 : s(t, h); }
};

// Every barrier alternates between two phases, so a waiter must not fall two
// behind.  The two sets of a row tile have barriers of their own: set j + 2 is
// not made before P V of set j is done, hence seen.
struct Ctl {
  uint64_t q_full, part[2], kv_full[10], kv_empty[10], s_full[2][2], p_ready[2][2], pv_done[2][2], o_done[2], fin[4];
  uint32_t tmem;
  int abort;
};

// All threads of the CTAs of a cluster, from whatever branch they are in.
__device__ __forceinline__ void cluster_join() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float peer_load(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// 8 columns of a row of the output, and what their rounding leaves out.
__device__ __forceinline__ void store_out(const float* o, __nv_bfloat16* out, __nv_bfloat16* rest) {
  uint4 w, e;
  uint32_t *u = &w.x, *f = &e.x;
#pragma unroll
  for (int c = 0; c < 4; ++c) u[c] = pack_bf16x2(o[2 * c], o[2 * c + 1]);
  *reinterpret_cast<uint4*>(out) = w;
  if (rest == nullptr) return;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    f[c] = pack_bf16x2(o[2 * c] - __uint_as_float(u[c] << 16), o[2 * c + 1] - __uint_as_float(u[c] & 0xffff0000u));
  *reinterpret_cast<uint4*>(rest) = e;
}


// SPLIT: the keys are divided among the CTAs of a cluster.  Each has a slice of
// whole streamed tiles and the same queries; at the end they read each other's
// row maxima and sums, put their weighted outputs into shared memory (where the
// ring was) and each adds up some of the columns, slices in order.
template <int DP, bool SPLIT>
__global__ void __launch_bounds__(Fwd<DP>::kThreads, DP == 64 ? 2 : 1)
    attention_fwd_tc(const Args a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using F = Fwd<DP>;
  constexpr int NT = F::NT, U = F::kUnit / kKeys;
  static_assert(NT * kRows * DP * 4 <= F::kStages * F::kTile);  // the weighted output of a slice
  extern __shared__ uint8_t smem_raw[];
  __shared__ Ctl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sbias = reinterpret_cast<float*>(smem + NT * F::kQTile + F::kStages * F::kTile);
  volatile int* abort = &ctl.abort;

  int tile;
  const int pack = a.pack, packs = a.heads / pack;
  const int n_slices = SPLIT ? a.splits : 1, block = blockIdx.x / n_slices, slice = blockIdx.x - block * n_slices;
  const Seq s = load_tile(a, block / packs, &tile);
  const int head0 = block % packs * pack, kv_head = head0 / (a.heads / a.kv_heads);
  const int r0 = tile * NT * kRows, off = s.lk - s.lq, total = s.lq * pack;
  // key tiles of each row tile
  int n_rows[NT], n_kv[NT], n_max = 0;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    n_rows[t] = min(kRows, max(0, total - r0 - t * kRows));
    const int last = (r0 + t * kRows + n_rows[t] - 1) / pack;  // its last query
    const int keys = n_rows[t] == 0 ? 0 : a.causal ? min(s.lk, last + off + 1) : s.lk;
    n_kv[t] = max(0, (keys + kKeys - 1) / kKeys);
    n_max = max(n_max, n_kv[t]);
  }
  auto units = [](int n) { return (n + U - 1) / U; };  // streamed tiles that hold n sets of 64 keys
  int key0 = 0;                                        // of the slice
  if (SPLIT) {
    const int per = (units(n_max) + n_slices - 1) / n_slices * U;
    key0 = slice * per * kKeys;
    n_max = max(0, min(per, n_max - slice * per));
#pragma unroll
    for (int t = 0; t < NT; ++t) n_kv[t] = max(0, min(per, n_kv[t] - slice * per));
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    ctl.abort = 0;
    mbar_init(&ctl.q_full, F::kSoftmax);
    mbar_init(&ctl.part[0], 1), mbar_init(&ctl.part[1], 1);
    for (int i = 0; i < F::kStages; ++i) mbar_init(&ctl.kv_full[i], 1), mbar_init(&ctl.kv_empty[i], NT);
    for (int t = 0; t < NT; ++t) {
      mbar_init(&ctl.o_done[t], 1);
      for (int h = 0; h < 2; ++h)
        mbar_init(&ctl.s_full[t][h], 1), mbar_init(&ctl.p_ready[t][h], kRows), mbar_init(&ctl.pv_done[t][h], 1);
    }
    for (int i = 0; i < 2 * NT; ++i) mbar_init(&ctl.fin[i], 1);
    fence_barrier_init();
  }
  if (warp == F::kMmaWarp) {
    tmem_alloc(&ctl.tmem, F::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(ctl.tmem), q_tile = uniform(smem_u32(smem)), kv_tile = q_tile + NT * F::kQTile;

  if (warp >= F::kLoadWarp) reg_dec<F::kOtherRegs>();
  if (warp == F::kLoadWarp) {
    // ---- loads: K and V tiles in turn
    TileLoader<DP> loader(ctl.part, abort);
    feed_ring<F::kStages>(loader, 2 * units(n_max), ctl.kv_full, ctl.kv_empty, abort, [&](int it, int st) {
      const int j = it >> 1;
      return loader.template load<F::kUnit>(kv_tile + st * F::kTile, it & 1 ? &v_map : &k_map, &ctl.kv_full[st], kv_head,
                                            s.k0 + key0 + j * F::kUnit, s.lk - key0 - j * F::kUnit);
    });
  } else if (warp >= F::kMmaWarp && warp < F::kMmaWarp + 2 * NT) {
    // ---- MMAs of row tile t
    if (n_max > 0) {
      const uint32_t leader = elect_lane();
      const int who = uniform(warp - F::kMmaWarp), t = who % NT, n_all = uniform(n_max), n = NT == 1 ? n_all : uniform(n_kv[t]);
      auto full = [&](int it) { return mbar_wait_warp(&ctl.kv_full[it % F::kStages], (it / F::kStages) & 1, abort); };
      // the last set of scores that uses its streamed tile
      auto last_of = [&](int j) { return j % U == U - 1 || j == n - 1; };
      bool ok = mbar_wait_warp(&ctl.q_full, 0, abort);
      int item;  // this warp's first streamed tile that only the other row tile uses
      if (who < NT) {
        const uint32_t idesc = idesc_bf16_f32(kRows, DP, false, true);
        for (int j = 0; j < n && ok; ++j) {
          const int it = 2 * (j / U) + 1, h = j & 1;
          if (!(ok = (j % U > 0 || full(it)) && mbar_wait_warp(&ctl.p_ready[t][h], (j >> 1) & 1, abort))) break;
          tc_fence_after();
          const uint32_t vd = desc_mn<F::kUnit>(kv_tile + (it % F::kStages) * F::kTile) + step_mn(j % U * (kKeys / 16));
#pragma unroll
          for (int i = 0; i < kKeys / 16; ++i)
            mma_ts(leader, tmem + F::o(t), tmem + F::p(t, h) + i * 8, vd + step_mn(i), idesc, j > 0 || i > 0);
          mma_commit(leader, &ctl.pv_done[t][h]);
          if (last_of(j)) mma_commit(leader, &ctl.kv_empty[it % F::kStages]);
        }
        mma_commit(leader, &ctl.o_done[t]);
        item = 2 * units(n) + 1;
      } else {
        const uint32_t idesc = idesc_bf16_f32(kRows, kKeys, false, false), qd = desc_k(q_tile + t * F::kQTile);
        for (int j = 0; j < n && ok; ++j) {
          const int it = 2 * (j / U), h = j & 1;
          if (j % U == 0 && !(ok = full(it))) break;
          // The scores of two sets before are read.  D = 128: they hold P by now, which P V has to be done with.
          if (j >= 2 && !(ok = mbar_wait_warp(DP == 64 ? &ctl.p_ready[t][h] : &ctl.pv_done[t][h], ((j >> 1) + 1) & 1, abort))) break;
          tc_fence_after();
          const uint32_t kd = desc_k(kv_tile + (it % F::kStages) * F::kTile) + j % U * (kKeys * 128 >> 4);
#pragma unroll
          for (int i = 0; i < DP / 16; ++i)
            mma_ss(leader, tmem + F::s(t, h), qd + step_k<kRows>(i), kd + step_k<F::kUnit>(i), idesc, i > 0);
          if (last_of(j)) mma_commit(leader, &ctl.kv_empty[it % F::kStages]);
          // D <= 64: the softmax writes P over that of two sets before, once P V is done with it
          if (DP == 64 && j >= 2 && !(ok = mbar_wait_warp(&ctl.pv_done[t][h], ((j >> 1) + 1) & 1, abort))) break;
          mma_commit(leader, &ctl.s_full[t][h]);
        }
        item = 2 * units(n);
      }
      for (; item < 2 * units(n_all) && ok; item += 2)
        if ((ok = full(item)) && leader) mbar_arrive(&ctl.kv_empty[item % F::kStages]);
      mma_commit(leader, &ctl.fin[who]);
      mbar_drain(&ctl.fin[who], 0);
    }
  } else if (warp < NT * 4) {
    reg_inc<F::kSoftmaxRegs>();
    // ---- softmax: thread = row
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const int r = r0 + t * kRows + row, n = NT == 1 ? n_max : n_kv[t], rows = NT == 1 ? n_rows[0] : n_rows[t];
    const bool valid = row < rows;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int tok = r / pack, pos = tok + off;
    const int limit = valid && a.causal ? min(s.lk, pos + 1) : s.lk;  // keys this row sees
    const float c2 = a.scale * kLog2e;
    BiasTable table;
    if (a.table != nullptr) table.begin(a, head0, pack, sbias, threadIdx.x, F::kSoftmax);
    load_tile_async<DP, kRows>(q_tile + t * F::kQTile,
                               static_cast<const __nv_bfloat16*>(a.q.p) + (int64_t)s.q0 * a.q.row + head0 * a.q.head, a.q.row,
                               a.q.head, pack, r0 + t * kRows, rows, a.dim, row);
    cp_async_commit();
    if (a.table != nullptr)
      table.finish<1>(a, head0, pack, sbias, sbias + pack * bias_stride(a.span), threadIdx.x, F::kSoftmax,
                      [] { named_bar_and(1, F::kSoftmax, true); });
    cp_async_wait<0>();
    fence_proxy_async_smem();
    mbar_arrive(&ctl.q_full);
    if (a.table != nullptr) named_bar_and(1, F::kSoftmax, true);
    const float* bias = sbias + (a.table != nullptr ? (r - tok * pack) * bias_stride(a.span) + a.span + kBiasPad : 0);
    // a far bias this large is added score by score, as the near ones are: see kDeep
    const bool large = a.table != nullptr && __any_sync(0xffffffffu, deep(bias[a.span]) || deep(bias[-a.span]));
    float m = -CUDART_INF_F, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int h = j & 1;
      if (!(ok = mbar_wait_warp(&ctl.s_full[t][h], (j >> 1) & 1, abort))) break;
      tc_fence_after();
      float x[kKeys];
#pragma unroll
      for (int c = 0; c < 2; ++c) tmem_ld32_issue(lanes + F::s(t, h) + c * 32, x + c * 32);
      tmem_wait_ld(x);
      const int k0 = key0 + j * kKeys;
      float mul = c2, add = 0.f;
      if (a.table != nullptr) {
        const int dist = pos - k0;  // to the first of the keys
        const bool far = dist - (kKeys - 1) >= a.span || dist <= -a.span;
        if (__all_sync(0xffffffffu, far) && !large) {
          add = dist > 0 ? bias[a.span] : bias[-a.span];
        } else {
          const float* b = bias + max(-a.span - kBiasPad + kKeys - 1, min(dist, a.span + kBiasPad));
#pragma unroll
          for (int c = 0; c < kKeys; ++c) x[c] = fmaf(x[c], c2, b[-c]);
          mul = 1.f;
        }
      }
      if (__any_sync(0xffffffffu, limit - k0 < kKeys)) {
        const int seen = limit - k0;
#pragma unroll
        for (int c = 0; c < kKeys; ++c) x[c] = c < seen ? x[c] : -CUDART_INF_F;
      }
      float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int c = 4; c + 1 < kKeys; c += 2) top[c / 2 & 3] = max3(top[c / 2 & 3], x[c], x[c + 1]);
      const float high = fmaf(max3(fmaxf(top[0], top[1]), top[2], top[3]), mul, add);
      if (__any_sync(0xffffffffu, high > m + kLazy)) {
        // some row's maximum moves: its sum and, once the last P V is done, its output follow
        const float m_new = fmaxf(m, high);
        const float fix = m == -CUDART_INF_F ? 0.f : ex2(m - m_new);
        m = m_new;
        l *= fix;
        if (j > 0) {
          if (!(ok = mbar_wait_warp(&ctl.pv_done[t][h ^ 1], ((j - 1) >> 1) & 1, abort))) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            float o[32];
            tmem_ld32_issue(lanes + F::o(t) + c * 32, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= fix;
            tmem_st32(lanes + F::o(t) + c * 32, reinterpret_cast<uint32_t*>(o));
          }
        }
      }
      const float base = add - (m == -CUDART_INF_F ? 0.f : m);  // a row without a visible key yet: 2^-inf = 0
      const uint64_t mul_2 = pair(mul, mul), base_2 = pair(base, base);
      uint64_t sum[2] = {0, 0};  // two pairs of float32 zeros
      uint32_t p[kKeys / 2];
#pragma unroll
      for (int c = 0; c < kKeys / 2; ++c) {
        float e0, e1;
        unpair(fma2(pair(x[2 * c], x[2 * c + 1]), mul_2, base_2), e0, e1);
        e0 = ex2(e0), e1 = ex2(e1);
        sum[c & 1] = add2(sum[c & 1], pair(e0, e1));
        p[c] = pack_bf16x2(e0, e1);
      }
      tmem_st32(lanes + F::p(t, h), p);
      float s0, s1;
      unpair(add2(sum[0], sum[1]), s0, s1);
      l += s0 + s1;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&ctl.p_ready[t][h]);
    }
    // ---- O / l, and the logarithm of the sum.  What follows writes over the queries: the products are done with them, or,
    // for a row tile without keys, every warp's copies of them have landed.
    if (ok) ok = mbar_wait_warp(n > 0 ? &ctl.o_done[t] : &ctl.q_full, 0, abort);
    tc_fence_after();
    const int head = head0 + (r - tok * pack);
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.o) + ((int64_t)(s.q0 + tok) * a.heads + head) * a.dim;
    __nv_bfloat16* rest =
        a.o_rest == nullptr ? nullptr : static_cast<__nv_bfloat16*>(a.o_rest) + ((int64_t)(s.q0 + tok) * a.heads + head) * a.dim;
    if (!SPLIT) {
      if (ok) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (valid && a.lse != nullptr) store_lse(a, (int64_t)head * a.tq + s.q0 + tok, m, l);
        // D = 128: in whole lines by way of shared memory, O first, what its rounding leaves out after another look at
        // tensor memory (one document of 8191 tokens: 264 us against 279 straight from the registers).  D <= 64: straight,
        // since the other CTA of the SM computes meanwhile (64 x 197 tokens: 79 us against 82 by way of shared memory).
        if constexpr (DP == 128) {
          const uint32_t stage = q_tile + t * F::kQTile + (warp & 3) * 32 * (DP * 2);  // the queries are done with
#pragma unroll 1
          for (int what = 0; what < (rest == nullptr ? 1 : 2); ++what) {
#pragma unroll 1
            for (int i = 0; i < DP / 32; ++i) {
              float o[32];
              __syncwarp();
              if (n > 0) {
                tmem_ld32_issue(lanes + F::o(t) + i * 32, o);
                tmem_wait_ld(o);
              }
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint32_t w[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  const float lo = l != 0.f ? o[q * 8 + 2 * c] * inv : 0.f, hi = l != 0.f ? o[q * 8 + 2 * c + 1] * inv : 0.f;
                  w[c] = pack_bf16x2(lo, hi);
                  if (what == 1) w[c] = pack_bf16x2(lo - __uint_as_float(w[c] << 16), hi - __uint_as_float(w[c] & 0xffff0000u));
                }
                stage_chunk<DP>(stage, i * 4 + q, w[0], w[1], w[2], w[3]);
              }
            }
            flush_rows<DP>(stage, what == 0 ? out : rest, valid, a.dim);
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < DP; i += 8) {
            float o[8] = {};
            __syncwarp();
            if (n > 0) {
              tmem_ld8_issue(lanes + F::o(t) + i, o);
              tmem_wait_ld(o);
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) o[c] = l != 0.f ? o[c] * inv : 0.f;
            if (valid && i < a.dim) store_out(o, out + i, rest == nullptr ? nullptr : rest + i);
          }
        }
      }
    } else {
      if (!ok || n == 0) m = -CUDART_INF_F, l = 0.f;
      const uint32_t stat = q_tile + t * F::kQTile + row * 8;  // the queries are done with
      asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(stat), "f"(m), "f"(l) : "memory");
      cluster_join();
      float high = -CUDART_INF_F, sum = 0.f;
      for (int p = 0; p < n_slices; ++p) high = fmaxf(high, peer_load(peer_addr(stat, p)));
      for (int p = 0; p < n_slices; ++p) {
        const float lp = peer_load(peer_addr(stat, p) + 4);
        if (lp != 0.f) sum = fmaf(lp, ex2(peer_load(peer_addr(stat, p)) - high), sum);
      }
      if (slice == 0 && valid && a.lse != nullptr) store_lse(a, (int64_t)head * a.tq + s.q0 + tok, high, sum);
      const float weight = l == 0.f ? 0.f : ex2(m - high) / sum;
      const uint32_t mine = kv_tile + t * DP * kRows * 4 + row * 4;  // (column, row): neighbouring lanes, neighbouring words
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        float o[32];
        __syncwarp();
        if (n > 0) {
          tmem_ld32_issue(lanes + F::o(t) + i * 32, o);
          tmem_wait_ld(o);
        }
#pragma unroll
        for (int c = 0; c < 32; ++c)
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + (i * 32 + c) * kRows * 4), "f"(l == 0.f ? 0.f : o[c] * weight) : "memory");
      }
      cluster_join();
      for (int c0 = slice * 8; c0 < a.dim; c0 += n_slices * 8) {
        float o[8] = {};
        for (int p = 0; p < n_slices; ++p) {
          const uint32_t from = peer_addr(mine, p) + c0 * kRows * 4;
#pragma unroll
          for (int c = 0; c < 8; ++c) o[c] += peer_load(from + c * kRows * 4);
        }
        if (valid) store_out(o, out + c0, rest == nullptr ? nullptr : rest + c0);
      }
      cluster_join();  // the others have read what is here
    }
    tc_fence_before();
  }
  if (SPLIT && warp >= NT * 4)
    for (int i = 0; i < 3; ++i) cluster_join();
  __syncthreads();
  if (warp == F::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, F::kCols);
  }
}

// Slices of the keys: as many, up to 8, as leave each 512 keys and an SM for each
// CTA.  16 queries of 12 heads of 64 over 4096 keys: 51 us in one slice, 35, 25
// and 21 in 2, 4 and 8; 129 queries of 32 heads of 128 on 8 key heads over 3129
// keys: 64, 45 and 33 (8 slices, more CTAs than SMs: 51).  512 keys in two slices
// gain nothing (64 CTAs with heads of 128: 22.5 us in one, 24.6 in two).
int split_count(const Args& a, int64_t ctas) {
  constexpr int kMaxSplits = 8, kMinKeys = 512;
  int s = 1;
  while (s < kMaxSplits && 2 * s * ctas <= 148 && 2 * s * kMinKeys <= a.longest) s *= 2;
  return s;
}

template <int DP, bool SPLIT>
int launch(const Args& a, int64_t ctas, cudaStream_t st) {
  const size_t smem = Fwd<DP>::kSmem + (a.table != nullptr ? a.pack * bias_floats(a.span, a.n_buckets) * sizeof(float) : 0);
  static SmemAllowed allowed;
  if (int rc = allow_smem(attention_fwd_tc<DP, SPLIT>, smem, allowed)) return rc;
  CUtensorMap k_map, v_map;
  const bool keys = a.tk > 0;  // without keys no tile is loaded
  if (int rc = make_tile_map(&k_map, keys ? a.k.p : a.q.p, keys ? a.tk : 1, keys ? a.kv_heads : 1, a.dim, a.k.row, a.k.head)) return rc;
  if (int rc = make_tile_map(&v_map, keys ? a.v.p : a.q.p, keys ? a.tk : 1, keys ? a.kv_heads : 1, a.dim, a.v.row, a.v.head)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(ctas * a.splits)), cfg.blockDim = dim3(Fwd<DP>::kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.splits, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = SPLIT ? 1 : 0;
  KF_CUDA_RET(cudaLaunchKernelEx(&cfg, attention_fwd_tc<DP, SPLIT>, a, k_map, v_map));
  return KF_OK;
}

template <int DP>
int launch(Args a, int n_tiles, cudaStream_t st) {
  const int64_t ctas = (int64_t)n_tiles * (a.heads / a.pack);
  a.splits = split_count(a, ctas);
  return a.splits > 1 ? launch<DP, true>(a, ctas, st) : launch<DP, false>(a, ctas, st);
}

}  // namespace

namespace attn {
int fwd_bf16(const Args& a, int n_tiles, cudaStream_t st) { return a.dim <= 64 ? launch<64>(a, n_tiles, st) : launch<128>(a, n_tiles, st); }
}  // namespace attn
}  // namespace kf
