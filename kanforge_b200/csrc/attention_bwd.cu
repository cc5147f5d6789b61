// Attention backward over packed sequences for bf16, on the tensor cores.
//
// Two kernels, so that every sum has one order without atomics: both form the
// scores again, P = 2^(t - lse), and dS = P (dP - delta) with dP = dO V^T.
//   dQ    rows = 128 queries of a head, walks over key tiles:
//         S, dP -> dS -> dQ += dS K; first it makes delta = dO . O, and it sums
//         dS by distance for the bias gradient.  The second kernel reads -delta
//         and -lse, which this one leaves in the workspace.
//   dK dV rows = 128 keys of a key head, walks over the query tiles of all heads
//         that share it: S^T, dP^T -> P^T, dS^T -> dV += P^T dO, dK += dS^T Q.
// Seven products of 128 x 128 x D a tile pair against five with one kernel;
// the five would add every dQ tile into memory in an order that varies.
// All scores live in tensor memory; P and dS go back there as bf16 (2^-9 of
// each term) and are the A operands of the products that sum them.  With D = 128 a
// CTA has an SM to itself; with D <= 64 two CTAs share one, so that one's chain of
// products and softmax runs under the other's.  Warps: softmax arithmetic (thread
// = row, 64 columns each), one that loads, and some that issue MMAs, one chain
// each.
//
// Measured, cold caches, causal: 8191 tokens, 16 heads of 128 on 4 key heads: dQ
// 0.37 ms (1.1 PFLOP/s), dK dV 0.63 ms (0.88 PFLOP/s; of 1.63 measured for bf16);
// 32 x 1024 tokens, 12 heads of 64 with a bias and its gradient: 0.26 ms (300 TFLOP/s)
// and 0.28 ms (370 TFLOP/s).  The chain S -> P -> dP -> dS -> product of a tile bounds
// them, of which tensor memory holds two an SM.  dK dV with four MMA warps (0.72 ms
// for the first) or with P and dS in columns of their own, one CTA an SM (0.69 ms,
// and 0.37 for the second) were slower.
#include "attention_tc.cuh"

namespace kf {
namespace {

using namespace attn;

template <int DP>
struct Bwd {
  static constexpr int kCols = DP == 64 ? 64 : 128;    // rows of a streamed tile, columns of the scores
  static constexpr int kStages = DP == 64 ? 6 : 4;     // streamed tiles in flight
  static constexpr int kFixed = tile_bytes<DP>(kRows), kTile = tile_bytes<DP>(kCols);
  static constexpr int kRing = 2 * kFixed, kFloats = kRing + kStages * kTile;  // byte offsets behind the fixed tiles
  static constexpr int kGroups = kCols / 64, kSoftmax = kGroups * 128;
  static constexpr int kLoadWarp = kGroups * 4, kMmaWarp = DP == 64 ? 5 : 10;
  static constexpr int kThreads = DP == 64 ? 256 : 384, kCtas = DP == 64 ? 2 : 1;
  // registers: 256 x 128 at launch = 128 x 192 + 128 x 64; 384 x 168 = 256 x 208 + 128 x 88
  static constexpr int kSoftmaxRegs = DP == 64 ? 192 : 208, kOtherRegs = DP == 64 ? 64 : 88;
  static constexpr uint32_t kTmem = DP == 64 ? 256 : 512;
};

// Every barrier alternates between two phases, so a waiter must not fall two
// behind: dS has a barrier for odd and one for even tiles, since the scores of
// the next tile are made before dS of this one is waited for.
struct Ctl {
  uint64_t fixed_full, part[2], full[8], empty[8], s_full, dp_full, s_read, ds_ready[2], dq_done, fin[2];
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ void init_barriers(Ctl* c, int stages, int softmax, int lane) {  // by a warp
  if (lane < stages) mbar_init(&c->full[lane], 1), mbar_init(&c->empty[lane], 1);
  if (lane < 2) mbar_init(&c->part[lane], 1), mbar_init(&c->ds_ready[lane], softmax), mbar_init(&c->fin[lane], 1);
  if (lane == 0) {
    c->abort = 0;
    mbar_init(&c->fixed_full, 2), mbar_init(&c->s_full, 1), mbar_init(&c->dp_full, 1), mbar_init(&c->dq_done, 1);
    mbar_init(&c->s_read, softmax);
  }
  fence_barrier_init();
}

// Barrier of the softmax warps.  A warp whose wait ran out calls it once with
// false and leaves; the others learn of it at their next call and leave too.
template <int DP>
__device__ __forceinline__ bool softmax_sync(bool ok = true) {
  return named_bar_and(1, Bwd<DP>::kSoftmax, ok);
}

// One row of a result: DP columns of this thread's lane times mul, dim of them stored.
template <int DP>
__device__ __forceinline__ void store_row(uint32_t lanes, __nv_bfloat16* out, int dim, float mul, bool zero, bool valid) {
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) {
    float o[32];
    __syncwarp();
    if (!zero) {
      tmem_ld32_issue(lanes + i * 32, o);
      tmem_wait_ld(o);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (!valid || i * 32 + q * 8 >= dim) continue;
      uint4 w;
      uint32_t* u = &w.x;
#pragma unroll
      for (int c = 0; c < 4; ++c) u[c] = zero ? 0u : pack_bf16x2(o[q * 8 + 2 * c] * mul, o[q * 8 + 2 * c + 1] * mul);
      *reinterpret_cast<uint4*>(out + i * 32 + q * 8) = w;
    }
  }
}

// The same in whole lines by way of `stage`, shared memory for 128 rows (the warp's
// 32 among them) that is free unless there was nothing to sum.  Faster for dQ (32 x
// 1024 tokens: 259 us, 266 straight from the registers) and slower for dK dV, whose
// two results follow each other (one document of 8191 tokens: 660 us, 628 straight).
template <int DP>
__device__ __forceinline__ void store_row_staged(uint32_t lanes, uint32_t stage, __nv_bfloat16* out, int dim, float mul, bool zero,
                                                 bool valid) {
  if (zero) {
    for (int c = 0; valid && c < dim; c += 8) *reinterpret_cast<uint4*>(out + c) = make_uint4(0, 0, 0, 0);
    return;
  }
  stage += (threadIdx.x >> 5 & 3) * 32 * (DP * 2);
#pragma unroll 1
  for (int i = 0; i < DP / 32; ++i) {
    float o[32];
    __syncwarp();
    tmem_ld32_issue(lanes + i * 32, o);
    tmem_wait_ld(o);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] = pack_bf16x2(o[q * 8 + 2 * c] * mul, o[q * 8 + 2 * c + 1] * mul);
      stage_chunk<DP>(stage, i * 4 + q, w[0], w[1], w[2], w[3]);
    }
  }
  flush_rows<DP>(stage, out, valid, dim);
}

// ---- dQ -------------------------------------------------------------------------
// Tensor memory: S, dP, dQ, two buffers of dS.
template <int DP>
struct QCols {
  static constexpr uint32_t s = 0, dp = Bwd<DP>::kCols, dq = 2 * Bwd<DP>::kCols, ds = dq + DP, ds_buffer = Bwd<DP>::kCols / 2;
};

// Floats behind the tiles: parts of delta, bias table, sums by distance of each
// block of 32 rows, block diagonals of each warp.
constexpr int kDiag = 48;                       // of a block of 32 x 16 scores: 47 diagonals
constexpr int kDiagWarp = 7 * kDiag + 32;       // four blocks, and what their unused stores reach
template <int DP>
__host__ __device__ constexpr int dq_floats(bool bias, bool grad, int span, int n_buckets) {
  static_assert(Bwd<DP>::kLoadWarp * kDiagWarp >= kMaxBuckets);
  return 2 * kRows + (bias ? bias_stride(span) : 0) +
         (grad ? 4 * (2 * span + 1) + Bwd<DP>::kLoadWarp * kDiagWarp : bias ? n_buckets : 0);
}

template <int DP>
__global__ void __launch_bounds__(Bwd<DP>::kThreads, Bwd<DP>::kCtas) attention_dq_tc(const Args a, const __grid_constant__ CUtensorMap q_map,
                                                               const __grid_constant__ CUtensorMap g_map,
                                                               const __grid_constant__ CUtensorMap k_map,
                                                               const __grid_constant__ CUtensorMap v_map) {
  using F = Bwd<DP>;
  using C = QCols<DP>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Ctl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sdelta = reinterpret_cast<float*>(smem + F::kFloats);  // (groups, 128) parts of delta
  float* sbias = sdelta + 2 * kRows;
  const int n_dist = 2 * a.span + 1;
  float* ssum = sbias + (a.table != nullptr ? bias_stride(a.span) : 0);  // (4, n_dist)
  float* sdiag = ssum + 4 * n_dist;                                      // (warps, kDiagWarp)
  float* column = a.dist_part != nullptr ? sdiag : ssum;  // of the learned table, needed before either is
  volatile int* abort = &ctl.abort;

  int tile;
  const Seq s = load_tile(a, blockIdx.x / a.heads, &tile);
  const int head = blockIdx.x % a.heads, kv_head = head / (a.heads / a.kv_heads);
  const int r0 = tile * kRows, off = s.lk - s.lq, n_rows = min(kRows, s.lq - r0);
  const int keys = a.causal ? max(0, min(s.lk, r0 + n_rows + off)) : s.lk;
  const int n = (keys + F::kCols - 1) / F::kCols;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool grad = a.dist_part != nullptr;

  if (warp == 0) init_barriers(&ctl, F::kStages, F::kSoftmax, lane);
  if (warp == F::kMmaWarp) {
    tmem_alloc(&ctl.tmem, F::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(ctl.tmem), q_tile = uniform(smem_u32(smem)), ring = q_tile + F::kRing;

  if (warp >= F::kLoadWarp) reg_dec<F::kOtherRegs>();
  if (warp == F::kLoadWarp) {
    // ---- loads: Q and dO, then K and V tiles in turn
    TileLoader<DP> loader(ctl.part, abort);
    if (loader.template load<kRows>(q_tile, &q_map, &ctl.fixed_full, head, s.q0 + r0, n_rows) &&
        loader.template load<kRows>(q_tile + F::kFixed, &g_map, &ctl.fixed_full, head, s.q0 + r0, n_rows))
      feed_ring<F::kStages>(loader, 2 * n, ctl.full, ctl.empty, abort, [&](int it, int st) {
        const int j = it >> 1;
        return loader.template load<F::kCols>(ring + st * F::kTile, it & 1 ? &v_map : &k_map, &ctl.full[st], kv_head,
                                              s.k0 + j * F::kCols, s.lk - j * F::kCols);
      });
    mbar_drain(&ctl.fixed_full, 0);
  } else if (warp >= F::kMmaWarp && warp < F::kMmaWarp + 2) {
    // ---- MMAs: one warp S, then dQ, the other dP.  S of the next tile goes ahead of dQ of this one.
    {
      const uint32_t leader = elect_lane();
      const int who = uniform(warp - F::kMmaWarp), n_all = uniform(n);
      const uint32_t idesc_s = idesc_bf16_f32(kRows, F::kCols, false, false), idesc_d = idesc_bf16_f32(kRows, DP, false, true);
      auto full = [&](int it) { return mbar_wait_warp(&ctl.full[it % F::kStages], (it / F::kStages) & 1, abort); };
      auto product = [&](int it, uint32_t d, uint32_t fixed, uint64_t* done) {
        tc_fence_after();
        const uint32_t ad = desc_k(fixed), bd = desc_k(ring + (it % F::kStages) * F::kTile);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) mma_ss(leader, d, ad + step_k<kRows>(i), bd + step_k<F::kCols>(i), idesc_s, i > 0);
        mma_commit(leader, done);
      };
      bool ok = mbar_wait_warp(&ctl.fixed_full, 0, abort);
      if (who == 0) {
        if (ok && n_all > 0 && (ok = full(0))) product(0, tmem + C::s, q_tile, &ctl.s_full);
        for (int j = 0; j < n_all && ok; ++j) {
          if (j + 1 < n_all) {
            if (!(ok = full(2 * (j + 1)) && mbar_wait_warp(&ctl.s_read, j & 1, abort))) break;
            product(2 * (j + 1), tmem + C::s, q_tile, &ctl.s_full);
          }
          if (!(ok = mbar_wait_warp(&ctl.ds_ready[j & 1], (j >> 1) & 1, abort))) break;
          tc_fence_after();
          const uint32_t kd = desc_mn<F::kCols>(ring + (2 * j % F::kStages) * F::kTile);
#pragma unroll
          for (int i = 0; i < F::kCols / 16; ++i)
            mma_ts(leader, tmem + C::dq, tmem + C::ds + (j & 1) * C::ds_buffer + i * 8, kd + step_mn(i), idesc_d, j > 0 || i > 0);
          mma_commit(leader, &ctl.empty[2 * j % F::kStages]);
        }
        mma_commit(leader, &ctl.dq_done);
      } else {
        for (int j = 0; j < n_all && ok; ++j) {
          if (!(ok = full(2 * j + 1) && (j == 0 || mbar_wait_warp(&ctl.ds_ready[(j - 1) & 1], ((j - 1) >> 1) & 1, abort)))) break;
          product(2 * j + 1, tmem + C::dp, q_tile + F::kFixed, &ctl.dp_full);
          mma_commit(leader, &ctl.empty[(2 * j + 1) % F::kStages]);
        }
      }
      mma_commit(leader, &ctl.fin[who]);
      mbar_drain(&ctl.fin[who], 0);
    }
  } else if (warp < F::kLoadWarp) {
    reg_inc<F::kSoftmaxRegs>();
    // ---- softmax arithmetic: thread = query, a warpgroup per half of a tile's keys
    BiasTable table;
    if (a.table != nullptr) table.begin(a, head, 1, sbias, threadIdx.x, F::kSoftmax);
    const int half = warp >> 2, row = (warp & 3) * 32 + lane, r = r0 + row;
    const bool valid = row < n_rows;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int pos = r + off;
    const int limit = valid && a.causal ? min(s.lk, pos + 1) : s.lk;
    const int64_t stat = (int64_t)head * a.tq + s.q0 + r;
    // delta = dO . O: D/8 lanes to a row, a warp has 32 rows or, with two warpgroups, 16 of them
    constexpr int LPR = DP / 8, RPP = 32 / LPR, PASSES = 32 / F::kGroups / RPP;
    {
      // all loads go out together; rows and columns that are not there read one that is
      const int c = lane % LPR * 8, first_row = (warp & 3) * 32 + half * 16 + lane / LPR, c_in = c < a.dim ? c : 0;
      const __nv_bfloat16* g = static_cast<const __nv_bfloat16*>(a.dout.p) + (int64_t)(s.q0 + r0) * a.dout.row + head * a.dout.head + c_in;
      const int64_t at = ((int64_t)(s.q0 + r0) * a.heads + head) * a.dim + c_in, o_row = (int64_t)a.heads * a.dim;
      const __nv_bfloat16 *o = static_cast<const __nv_bfloat16*>(a.o) + at, *e = static_cast<const __nv_bfloat16*>(a.o_rest) + at;
      uint4 gv[PASSES], ov[PASSES], ev[PASSES];
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int64_t from = min(first_row + i * RPP, n_rows - 1);
        gv[i] = *reinterpret_cast<const uint4*>(g + from * a.dout.row);
        ov[i] = *reinterpret_cast<const uint4*>(o + from * o_row);
        ev[i] = *reinterpret_cast<const uint4*>(e + from * o_row);
      }
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const uint32_t *gw = &gv[i].x, *ow = &ov[i].x, *ew = &ev[i].x;
        float d = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          d = fmaf(__uint_as_float(gw[k] << 16), __uint_as_float(ow[k] << 16) + __uint_as_float(ew[k] << 16), d);
          d = fmaf(__uint_as_float(gw[k] & 0xffff0000u), __uint_as_float(ow[k] & 0xffff0000u) + __uint_as_float(ew[k] & 0xffff0000u), d);
        }
        if (c >= a.dim) d = 0.f;
#pragma unroll
        for (int k = LPR / 2; k > 0; k >>= 1) d += __shfl_xor_sync(0xffffffffu, d, k);
        if (lane % LPR == 0) sdelta[first_row + i * RPP] = d;
      }
    }
    if (grad)
      for (int i = threadIdx.x; i < 4 * n_dist; i += F::kSoftmax) ssum[i] = 0.f;
    if (a.table != nullptr) table.finish<0>(a, head, 1, sbias, column, threadIdx.x, F::kSoftmax, [] { softmax_sync<DP>(); });
    softmax_sync<DP>();
    float delta = sdelta[row];
    if (F::kGroups == 2) softmax_sync<DP>();  // sdelta is written again below
    // O carries the rounding of P, which weighs most where a row sees few keys:
    // rows whose keys all lie in the first tile get delta = sum P dP there.
    const bool short_rows = (a.causal ? r0 + off + 1 : s.lk) <= F::kCols;
    if (valid && half == 0 && !(short_rows && n > 0)) a.delta[stat] = -delta;
    // a row that sees one key has dS = 0; rows past the sequence likewise
    const float lse_row = valid ? a.lse[stat] : 0.f, lse = valid && !one_key(a, s, pos) ? lse_row : CUDART_INF_F;
    if (valid && half == 0) a.delta[(int64_t)a.heads * a.tq + stat] = -lse_row;
    const bool large = a.table != nullptr && __any_sync(0xffffffffu, deep(lse_row));  // see kDeep
    if (valid && half == 0 && lane == 0) a.delta[2 * (int64_t)a.heads * a.tq + stat] = large ? 1.f : 0.f;
    const float c2 = a.scale * kLog2e;
    const float* bias = sbias + a.span + kBiasPad;
    float far_sum[2] = {0.f, 0.f};  // dS at distances >= span, <= -span
    // Sum over the keys P dP = dO . O only as far as O's P was rounded, while a row's dS add up to 0: what they do
    // add up to goes off the sums of the tiles beyond the span, by the share of P there.  Elsewhere the keys of a
    // bucket are too few for it to show.
    float row_sum = 0.f, far_p[2] = {0.f, 0.f};
    auto sum64 = [](const float (&v)[64]) {
      uint64_t t[4] = {pair(v[0], v[1]), pair(v[2], v[3]), pair(v[4], v[5]), pair(v[6], v[7])};
#pragma unroll
      for (int i = 8; i < 64; i += 2) t[i / 2 & 3] = add2(t[i / 2 & 3], pair(v[i], v[i + 1]));
      return sum_of(add2(add2(t[0], t[1]), add2(t[2], t[3])));
    };
    bool ok = true, together = true, owed = F::kGroups == 2 && short_rows && n > 0;  // owed: the barrier of delta is still ahead
    for (int j = 0; j < n; ++j) {
      if (!(ok = mbar_wait_warp(&ctl.s_full, j & 1, abort))) break;
      tc_fence_after();
      float x[64];
#pragma unroll
      for (int i = 0; i < 2; ++i) tmem_ld32_issue(lanes + C::s + half * 64 + i * 32, x + i * 32);
      tmem_wait_ld(x);
      tc_fence_before();
      mbar_arrive(&ctl.s_read);
      const int k0 = j * F::kCols + half * 64;
      const int dist = pos - k0;
      bool near = false;
      float base = -lse;
      if (a.table != nullptr) {
        near = !__all_sync(0xffffffffu, dist - 63 >= a.span || dist <= -a.span) || large;
        if (near) {
          const float* b = bias + max(-a.span - kBiasPad + 63, min(dist, a.span + kBiasPad));
          const float minus = large ? 0.f : lse;
#pragma unroll
          for (int i = 0; i < 64; ++i) x[i] = fmaf(x[i], c2, b[-i] - minus);
        } else {
          base = (dist > 0 ? bias[a.span] : bias[-a.span]) - lse;
        }
      }
      if (!near) {
        const uint64_t c2_2 = pair(c2, c2), base_2 = pair(base, base);
#pragma unroll
        for (int i = 0; i < 64; i += 2) unpair(fma2(pair(x[i], x[i + 1]), c2_2, base_2), x[i], x[i + 1]);
      }
      if (large) {
        const float minus = near ? lse : 0.f, rest = valid ? load_lse_rest(a, stat) : 0.f;
#pragma unroll
        for (int i = 0; i < 64; ++i) x[i] = (x[i] - minus) - rest;
      }
#pragma unroll
      for (int i = 0; i < 64; ++i) x[i] = ex2(x[i]);
      const bool masked = __any_sync(0xffffffffu, limit - k0 < 64);
      const int d0 = r0 + off - j * F::kCols;  // distance of the tile's first query and key
      const bool far = d0 - (F::kCols - 1) >= a.span || d0 + kRows - 1 <= -a.span;  // farther than the span from all its keys
      if (grad && far && !masked) far_p[d0 > 0 ? 0 : 1] += sum64(x);
      if (!(ok = mbar_wait_warp(&ctl.dp_full, j & 1, abort))) break;
      tc_fence_after();
      const int seen = limit - k0;
      if (short_rows && j == 0) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float d[32];
          tmem_ld32_issue(lanes + C::dp + half * 64 + h * 32, d);
          tmem_wait_ld(d);
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[i & 3] += h * 32 + i < seen ? x[h * 32 + i] * d[i] : 0.f;
        }
        float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (F::kGroups == 2) {
          sdelta[half * kRows + row] = all;
          if (!(together = softmax_sync<DP>())) break;
          owed = false;
          all = sdelta[row] + sdelta[kRows + row];
        }
        if (limit <= F::kCols) delta = all;
        if (valid && half == 0) a.delta[stat] = -delta;
      }
      const uint64_t minus_delta = pair(-delta, -delta);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float d[32];
        tmem_ld32_issue(lanes + C::dp + half * 64 + h * 32, d);
        tmem_wait_ld(d);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float *x0 = &x[h * 32 + i], *x1 = x0 + 1;
          unpair(mul2(pair(*x0, *x1), add2(pair(d[i], d[i + 1]), minus_delta)), *x0, *x1);
        }
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < 64; ++i) x[i] = i < seen ? x[i] : 0.f;
      }
      uint32_t w[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
      tmem_st32(lanes + C::ds + (j & 1) * C::ds_buffer + half * 32, w);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&ctl.ds_ready[j & 1]);
      if (!grad) continue;
      // ---- the bias gradient.  A far tile adds to one bucket.
      const float sum = sum64(x);
      row_sum += sum;
      if (far) {
        far_sum[d0 > 0 ? 0 : 1] += sum;
      } else {
        // A partial sum moves along its diagonal, one lane up for each column; lane 31's is complete.
        // Four blocks of 32 rows x 16 columns at a time, to have four such chains in flight.
        // The other lanes store beside it what nothing reads: a store by one lane would be a branch.
        const float keep = lane == 0 ? 0.f : 1.f;
        float* out = sdiag + warp * kDiagWarp;  // of block h: index row - column + 15
        float* put = lane == 31 ? out + 46 : out + 4 * kDiag + lane;
        const int back = lane == 31 ? 1 : 0;
        float acc[4];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            acc[h] = c == 0 ? x[h * 16] : fmaf(__shfl_up_sync(0xffffffffu, acc[h], 1), keep, x[h * 16 + c]);
            put[h * kDiag] = acc[h];
          }
          put -= back;
        }
        if (lane < 31) {
#pragma unroll
          for (int h = 0; h < 4; ++h) out[h * kDiag + lane] = acc[h];
        }
        __syncwarp();
        // The warp adds its 95 diagonals to the sums of its 32 rows, which with two warpgroups it
        // shares with one other warp: that one's turn comes after a barrier.
        if (F::kGroups == 2 && half == 1 && !(together = softmax_sync<DP>())) break;
        float* sums = ssum + (warp & 3) * n_dist + a.span;
        const int dw = d0 + (warp & 3) * 32 - half * 64;  // distance of the warp's first row and column
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const int i = k * 32 + lane - 63;  // row - column
          float sum = 0.f;
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int e = i + h * 16 + 15;
            if (e >= 0 && e < 47) sum += out[h * kDiag + e];
          }
          const int dd = dw + i;
          if (dd >= a.span)
            far_sum[0] += sum;
          else if (dd <= -a.span)
            far_sum[1] += sum;
          else
            sums[dd] += sum;
        }
        __syncwarp();
        if (F::kGroups == 2) {
          if (half == 0 && !(together = softmax_sync<DP>())) break;
          if (!(together = softmax_sync<DP>())) break;
        }
      }
    }
    if (ok && together && n > 0) ok = mbar_wait_warp(&ctl.dq_done, 0, abort);
    if ((grad || owed) && together) together = softmax_sync<DP>(ok);
    if (ok && together) {
      tc_fence_after();
      if (half == 0)
        store_row_staged<DP>(lanes + C::dq, q_tile, static_cast<__nv_bfloat16*>(a.dq) + ((int64_t)(s.q0 + r) * a.heads + head) * a.dim, a.dim,
                      a.scale, n == 0, valid);
      if (grad) {
        if (F::kGroups == 2) {
          sdelta[half * kRows + row] = row_sum;
          softmax_sync<DP>();
          row_sum = sdelta[row] + sdelta[kRows + row];
        }
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          far_sum[f] -= row_sum * far_p[f];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) far_sum[f] += __shfl_xor_sync(0xffffffffu, far_sum[f], o);
          if (lane == 0) sdiag[f * 8 + warp] = far_sum[f];
        }
        softmax_sync<DP>();  // the sums of all warps, too
        float* out = a.dist_part + (int64_t)blockIdx.x * n_dist;
        for (int e = threadIdx.x; e < n_dist; e += F::kSoftmax) {
          float sum = (ssum[e] + ssum[n_dist + e]) + (ssum[2 * n_dist + e] + ssum[3 * n_dist + e]);
          if (e == 0 || e == 2 * a.span) {
            const float* far = sdiag + (e == 0 ? 8 : 0);
            for (int w = 0; w < F::kLoadWarp; ++w) sum += far[w];
          }
          out[e] = sum;
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == F::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, F::kTmem);
  }
}

// ---- dK, dV -----------------------------------------------------------------------
// A tile of 64 queries is one warpgroup's.  With D = 128 two warpgroups take the
// tiles in turn, so that one's softmax runs under the products of the other's
// tile; with D <= 64 the other CTA of the SM does that.  Tensor memory: S^T and dP^T
// of each group, dV, dK.  P^T and dS^T lie in their scores' columns, and the next
// scores of the group wait for the product that reads them.  The MMA warps: one
// makes S^T and dP^T, one dV, one dK.
template <int DP>
struct Kv {
  static constexpr int kGroups = DP == 64 ? 1 : 2, kCols = 64;
  static constexpr int kStages = DP == 64 ? 6 : 8;
  static constexpr int kFixed = tile_bytes<DP>(kRows), kTile = tile_bytes<DP>(kCols);
  static constexpr int kRing = 2 * kFixed, kFloats = kRing + kStages * kTile;
  static constexpr int kLoadWarp = kGroups * 4, kMmaWarp = kLoadWarp + 1;
  static constexpr int kThreads = kGroups * 128 + 128, kCtas = DP == 64 ? 2 : 1;
  // registers: 256 x 128 at launch = 128 x 192 + 128 x 64; 384 x 168 = 256 x 208 + 128 x 88
  static constexpr int kSoftmaxRegs = DP == 64 ? 192 : 208, kOtherRegs = DP == 64 ? 64 : 88;
  static constexpr uint32_t kTmem = DP == 64 ? 256 : 512;
  __device__ static constexpr uint32_t s(int g) { return g * kCols; }
  __device__ static constexpr uint32_t dp(int g) { return (kGroups + g) * kCols; }
  static constexpr uint32_t dv = 2 * kGroups * kCols, dk = dv + DP;
};

struct KvCtl {
  uint64_t fixed_full, part[2], full[8], empty[8], stat_full[8];
  uint64_t s_full[2], dp_full[2], p_ready[2], ds_ready[2], dv_done[2], dk_done[2], dv_all, dk_all, fin;
  uint32_t tmem;
  int abort;
};

template <int DP>
__host__ __device__ constexpr int dkdv_floats(bool bias, int span, int n_buckets) {
  return Kv<DP>::kStages * 2 * Kv<DP>::kCols + (bias ? Kv<DP>::kGroups * bias_floats(span, n_buckets) : 0);
}

template <int DP, bool BIAS>
__global__ void __launch_bounds__(Kv<DP>::kThreads, Kv<DP>::kCtas)
    attention_dkdv_tc(const Args a, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap g_map,
                      const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using F = Kv<DP>;
  constexpr int G = F::kGroups;
  extern __shared__ uint8_t smem_raw[];
  __shared__ KvCtl ctl;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sstat = reinterpret_cast<float*>(smem + F::kFloats);  // -lse, -delta of each stage in the ring
  volatile int* abort = &ctl.abort;

  int tile;
  const Seq s = load_tile(a, blockIdx.x / a.kv_heads, &tile);
  const int kv_head = blockIdx.x % a.kv_heads, group = a.heads / a.kv_heads;
  const int r0 = tile * kRows, off = s.lk - s.lq, n_rows = min(kRows, s.lk - r0);
  const int first = a.causal ? max(0, r0 - off) / F::kCols : 0;  // earlier query tiles see none of these keys
  const int per_head = max(0, (s.lq + F::kCols - 1) / F::kCols - first), n = group * per_head;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    ctl.abort = 0;
    mbar_init(&ctl.fixed_full, 2);
    mbar_init(&ctl.part[0], 1), mbar_init(&ctl.part[1], 1);
    for (int i = 0; i < F::kStages; ++i) mbar_init(&ctl.full[i], 1), mbar_init(&ctl.empty[i], 2), mbar_init(&ctl.stat_full[i], 32);
    for (int g = 0; g < G; ++g) {
      mbar_init(&ctl.s_full[g], 1), mbar_init(&ctl.dp_full[g], 1), mbar_init(&ctl.dv_done[g], 1), mbar_init(&ctl.dk_done[g], 1);
      mbar_init(&ctl.p_ready[g], 128), mbar_init(&ctl.ds_ready[g], 128);
    }
    mbar_init(&ctl.dv_all, 1), mbar_init(&ctl.dk_all, 1), mbar_init(&ctl.fin, 1);
    fence_barrier_init();
  }
  if (warp == F::kMmaWarp) {
    tmem_alloc(&ctl.tmem, F::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(ctl.tmem), k_tile = uniform(smem_u32(smem)), ring = k_tile + F::kRing;

  if (warp >= F::kLoadWarp) reg_dec<F::kOtherRegs>();
  if (warp == F::kLoadWarp) {
    // ---- loads: K and V, then Q (with -lse and -delta) and dO tiles in turn
    TileLoader<DP> loader(ctl.part, abort);
    if (loader.template load<kRows>(k_tile, &k_map, &ctl.fixed_full, kv_head, s.k0 + r0, n_rows) &&
        loader.template load<kRows>(k_tile + F::kFixed, &v_map, &ctl.fixed_full, kv_head, s.k0 + r0, n_rows))
      feed_ring<F::kStages>(loader, 2 * n, ctl.full, ctl.empty, abort, [&](int it, int st) {
        const int i = it >> 1, head = kv_head * group + i / per_head, q0 = (first + i % per_head) * F::kCols;
        const int n_q = min(F::kCols, s.lq - q0);
        if (!(it & 1)) {
          const int64_t stat = (int64_t)head * a.tq + s.q0 + q0;
          for (int c = lane; c < 2 * F::kCols; c += 32) {
            const int col = c & (F::kCols - 1);
            const bool in = col < n_q;
            const float* f = a.delta + (c < F::kCols ? (int64_t)a.heads * a.tq : 0) + stat + (in ? col : 0);
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(sstat + st * 2 * F::kCols + c)), "l"(f),
                         "r"(in ? 4 : 0)
                         : "memory");
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&ctl.stat_full[st])) : "memory");
        }
        return loader.template load<F::kCols>(ring + st * F::kTile, it & 1 ? &g_map : &q_map, &ctl.full[st], head, s.q0 + q0, n_q);
      });
    cp_async_wait<0>();
    mbar_drain(&ctl.fixed_full, 0);
  } else if (warp >= F::kMmaWarp) {
    // ---- MMAs
    {
      const uint32_t leader = elect_lane();
      const int role = uniform(warp - F::kMmaWarp), n_all = uniform(n);
      auto full = [&](int it) { return mbar_wait_warp(&ctl.full[it % F::kStages], (it / F::kStages) & 1, abort); };
      bool ok = mbar_wait_warp(&ctl.fixed_full, 0, abort);
      if (role == 0) {
        const uint32_t idesc = idesc_bf16_f32(kRows, F::kCols, false, false), kd = desc_k(k_tile), vd = desc_k(k_tile + F::kFixed);
        auto product = [&](int it, uint32_t d, uint32_t fixed, uint64_t* made) {
          tc_fence_after();
          const uint32_t bd = desc_k(ring + (it % F::kStages) * F::kTile);
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) mma_ss(leader, d, fixed + step_k<kRows>(c), bd + step_k<F::kCols>(c), idesc, c > 0);
          mma_commit(leader, made);
          mma_commit(leader, &ctl.empty[it % F::kStages]);
        };
        for (int i = 0; i < n_all && ok; ++i) {
          const int g = i % G;
          const uint32_t before = (i / G - 1) & 1;  // phase of the group's tile before
          if (!(ok = full(2 * i) && (i < G || mbar_wait_warp(&ctl.dv_done[g], before, abort)))) break;
          product(2 * i, tmem + F::s(g), kd, &ctl.s_full[g]);
          if (!(ok = full(2 * i + 1) && (i < G || mbar_wait_warp(&ctl.dk_done[g], before, abort)))) break;
          product(2 * i + 1, tmem + F::dp(g), vd, &ctl.dp_full[g]);
        }
        mma_commit(leader, &ctl.fin);
        mbar_drain(&ctl.fin, 0);
      } else {
        const bool v = role == 1;  // dV takes dO, dK takes Q
        const uint32_t idesc = idesc_bf16_f32(kRows, DP, false, true), acc = tmem + (v ? F::dv : F::dk);
        for (int i = 0; i < n_all && ok; ++i) {
          const int g = i % G, it = 2 * i + v;
          // the tile is there long before: its barrier is looked at first, off the way from softmax to product
          if (!(ok = full(it) && mbar_wait_warp(v ? &ctl.p_ready[g] : &ctl.ds_ready[g], (i / G) & 1, abort))) break;
          tc_fence_after();
          const uint32_t bd = desc_mn<F::kCols>(ring + (it % F::kStages) * F::kTile), p = tmem + (v ? F::s(g) : F::dp(g));
#pragma unroll
          for (int c = 0; c < F::kCols / 16; ++c) mma_ts(leader, acc, p + c * 8, bd + step_mn(c), idesc, i > 0 || c > 0);
          mma_commit(leader, v ? &ctl.dv_done[g] : &ctl.dk_done[g]);
          mma_commit(leader, &ctl.empty[it % F::kStages]);
        }
        uint64_t* all = v ? &ctl.dv_all : &ctl.dk_all;
        mma_commit(leader, all);
        mbar_drain(all, 0);
      }
    }
  } else {
    reg_inc<F::kSoftmaxRegs>();
    // ---- softmax arithmetic: thread = key
    const int g = warp >> 2, row = (warp & 3) * 32 + lane, key = r0 + row;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float c2 = a.scale * kLog2e;
    float* sbias = sstat + F::kStages * 2 * F::kCols + g * bias_floats(a.span, a.n_buckets);
    const float* bias = sbias + a.span + kBiasPad;
    // barrier of the group: see softmax_sync
    auto group_sync = [&](bool ok) { return named_bar_and(1 + g, 128, ok); };
    bool ok = true, together = true;
    int head_in = -1;  // whose bias table is there
    // Whether any row of the group's heads is beyond kDeep: what dQ left for every 32 rows.  (A look at each tile's
    // statistics instead costs its chain up to 15%, this 1.5 to 3%, for which calls without a bias have a kernel
    // of their own: 16 packed documents 141 us, with both in one 151.)
    bool large = false;
    for (int h = 0; BIAS && a.lse_rest && h < group; ++h)
      for (int q = lane * 32; q < s.lq; q += 32 * 32) large |= a.delta[2 * (int64_t)a.heads * a.tq + (int64_t)(kv_head * group + h) * a.tq + s.q0 + q] != 0.f;
    if (BIAS) large = __any_sync(0xffffffffu, large);
    for (int i = g; i < n; i += G) {
      const int st = 2 * i % F::kStages, q0 = (first + i % per_head) * F::kCols, head = kv_head * group + i / per_head;
      const uint32_t phase = (i / G) & 1;
      if (BIAS && head != head_in) {
        head_in = head;
        if (!(together = group_sync(true))) break;
        expand_bias(a, head, 1, sbias, sbias + bias_stride(a.span), threadIdx.x & 127, 128, [&] { together = group_sync(true); });
        if (!together || !(together = group_sync(true))) break;
      }
      ok = mbar_wait_warp(&ctl.stat_full[st], (2 * i / F::kStages) & 1, abort) && mbar_wait_warp(&ctl.s_full[g], phase, abort);
      if (!ok) break;
      tc_fence_after();
      float x[F::kCols];
#pragma unroll
      for (int h = 0; h < 2; ++h) tmem_ld32_issue(lanes + F::s(g) + h * 32, x + h * 32);
      tmem_wait_ld(x);
      const ulonglong2* lse = reinterpret_cast<const ulonglong2*>(sstat + st * 2 * F::kCols);  // pairs of -lse
      const ulonglong2* delta = lse + F::kCols / 4;
      const int dist = q0 + off - key;  // of the first column
      float mul = c2, add = 0.f;
      if (BIAS) {
        if (__all_sync(0xffffffffu, dist >= a.span || dist + F::kCols - 1 <= -a.span) && !large) {
          add = dist > 0 ? bias[a.span] : bias[-a.span];
        } else {
          const float* b = bias + max(-a.span - kBiasPad, min(dist, a.span + kBiasPad - F::kCols + 1));
#pragma unroll
          for (int c = 0; c < F::kCols; ++c) x[c] = fmaf(x[c], c2, b[c]);
          mul = 1.f;
        }
      }
      const uint64_t mul_2 = pair(mul, mul), add_2 = pair(add, add);
#pragma unroll
      for (int c = 0; c < F::kCols; c += 4) {
        const ulonglong2 e = lse[c / 4];
        unpair(fma2(pair(x[c], x[c + 1]), mul_2, add2(add_2, e.x)), x[c], x[c + 1]);
        unpair(fma2(pair(x[c + 2], x[c + 3]), mul_2, add2(add_2, e.y)), x[c + 2], x[c + 3]);
      }
#pragma unroll
      for (int c = 0; c < F::kCols; ++c) x[c] = ex2(x[c]);
      // columns of queries that see this key: [from, to)
      const int from = a.causal ? key - off - q0 : 0, to = s.lq - q0;
      const bool masked = __any_sync(0xffffffffu, from > 0 || to < F::kCols || s.lk == 1 || (a.causal && q0 + off <= 0)) || large;
      if (masked) {
        if (large) {  // the scores are their row's maximum or far below it: what is left of lse is a factor
          const int64_t at = (int64_t)head * a.tq + s.q0 + q0 + lane;
#pragma unroll
          for (int h = 0; h < F::kCols / 32; ++h) {
            const float f = q0 + h * 32 + lane < s.lq ? ex2(-load_lse_rest(a, at + h * 32)) : 0.f;
#pragma unroll
            for (int c = 0; c < 32; ++c) x[h * 32 + c] *= __shfl_sync(0xffffffffu, f, c);
          }
        }
#pragma unroll
        for (int c = 0; c < F::kCols; ++c) x[c] = c >= from && c < to ? x[c] : 0.f;
      }
      uint32_t w[F::kCols / 2];
#pragma unroll
      for (int c = 0; c < F::kCols / 2; ++c) w[c] = pack_bf16x2(x[2 * c], x[2 * c + 1]);
      tmem_st32(lanes + F::s(g), w);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&ctl.p_ready[g]);

      if (!(ok = mbar_wait_warp(&ctl.dp_full[g], phase, abort))) break;
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float d[32];
        tmem_ld32_issue(lanes + F::dp(g) + h * 32, d);
        tmem_wait_ld(d);
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const ulonglong2 e = delta[(h * 32 + c) / 4];  // pairs of -delta
          float* y = &x[h * 32 + c];
          unpair(mul2(pair(y[0], y[1]), add2(pair(d[c], d[c + 1]), e.x)), y[0], y[1]);
          unpair(mul2(pair(y[2], y[3]), add2(pair(d[c + 2], d[c + 3]), e.y)), y[2], y[3]);
        }
      }
      if (masked) {
        const int one = a.causal ? -off - q0 : -1;  // the query that sees one key
#pragma unroll
        for (int c = 0; c < F::kCols; ++c) x[c] = c >= from && c < to && c != one && s.lk > 1 ? x[c] : 0.f;
      }
#pragma unroll
      for (int c = 0; c < F::kCols / 2; ++c) w[c] = pack_bf16x2(x[2 * c], x[2 * c + 1]);
      tmem_st32(lanes + F::dp(g), w);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&ctl.ds_ready[g]);
    }
    if (BIAS && together) together = group_sync(ok);
    if (ok && together && n > 0) ok = mbar_wait_warp(&ctl.dv_all, 0, abort) && mbar_wait_warp(&ctl.dk_all, 0, abort);
    if (ok && together) {
      tc_fence_after();
      const int64_t at = ((int64_t)(s.k0 + key) * a.kv_heads + kv_head) * a.dim;
      if (g == 0) store_row<DP>(lanes + F::dv, static_cast<__nv_bfloat16*>(a.dv) + at, a.dim, 1.f, n == 0, row < n_rows);
      if (g == G - 1) store_row<DP>(lanes + F::dk, static_cast<__nv_bfloat16*>(a.dk) + at, a.dim, a.scale, n == 0, row < n_rows);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == F::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, F::kTmem);
  }
}

template <int DP>
int launch(const Args& a0, const Tile* k_tiles, int n_q, int n_k, cudaStream_t st) {
  Args a = a0;
  const bool bias = a.table != nullptr;
  // a side without rows has no tiles, but the map of its tensor must be valid
  auto map = [&](CUtensorMap* m, const Strided& t, int64_t rows, int heads) {
    return rows > 0 ? make_tile_map(m, t.p, rows, heads, a.dim, t.row, t.head)
                    : make_tile_map(m, n_q > 0 ? a.q.p : a.k.p, 1, 1, a.dim, 0, 0);
  };
  CUtensorMap q_map, g_map, k_map, v_map;
  if (int rc = map(&q_map, a.q, a.tq, a.heads)) return rc;
  if (int rc = map(&g_map, a.dout, a.tq, a.heads)) return rc;
  if (int rc = map(&k_map, a.k, a.tk, a.kv_heads)) return rc;
  if (int rc = map(&v_map, a.v, a.tk, a.kv_heads)) return rc;
  if (n_q > 0) {
    const size_t smem = 1024 + Bwd<DP>::kFloats + dq_floats<DP>(bias, a.dist_part != nullptr, a.span, a.n_buckets) * sizeof(float);
    static SmemAllowed allowed;
    if (int rc = allow_smem(attention_dq_tc<DP>, smem, allowed)) return rc;
    attention_dq_tc<DP><<<(unsigned)n_q * a.heads, Bwd<DP>::kThreads, smem, st>>>(a, q_map, g_map, k_map, v_map);
    if (int rc = check_launch("kf_attention_bwd")) return rc;
  }
  if (n_k > 0) {
    a.tiles = k_tiles;
    const size_t smem = 1024 + Kv<DP>::kFloats + dkdv_floats<DP>(bias, a.span, a.n_buckets) * sizeof(float);
    static SmemAllowed allowed, allowed_bias;
    auto* kernel = bias ? attention_dkdv_tc<DP, true> : attention_dkdv_tc<DP, false>;
    if (int rc = allow_smem(kernel, smem, bias ? allowed_bias : allowed)) return rc;
    kernel<<<(unsigned)n_k * a.kv_heads, Kv<DP>::kThreads, smem, st>>>(a, q_map, g_map, k_map, v_map);
    return check_launch("kf_attention_bwd");
  }
  return KF_OK;
}

}  // namespace

namespace attn {
int bwd_bf16(const Args& a, const Tile* k_tiles, int n_q, int n_k, cudaStream_t st) {
  if (n_q == 0 && n_k == 0) return KF_OK;
  return a.dim <= 64 ? launch<64>(a, k_tiles, n_q, n_k, st) : launch<128>(a, k_tiles, n_q, n_k, st);
}
}  // namespace attn
}  // namespace kf
