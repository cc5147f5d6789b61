// What the attention kernels share: the packed sequences, the launch operands
// and the learned relative position bias.
//
// Query i of a sequence with Lq queries and Lk keys stands at position
// i + Lk - Lq; with d = position - key, scores are kept in base 2:
//   t = scale log2(e) q.k + log2(e) B[bucket(d), head],  P = 2^(t - lse),
// and lse = max + log2(sum) is what the forward keeps for the backward.
#pragma once

#include <math_constants.h>

#include <initializer_list>

#include "common.cuh"

namespace kf {
namespace attn {

constexpr int kMaxDim = 128;
constexpr int kMaxSpan = 512;    // largest distance with a bias of its own
constexpr int kMaxBuckets = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct Seq {
  int q0, lq, k0, lk;  // rows of the queries, of the keys
};

struct __align__(16) Tile {
  Seq s;
  int index;  // of the tile in its sequence
  int unused[3];
};

struct Strided {  // (tokens, heads, dim), last dimension contiguous; strides in elements
  const void* p;
  int64_t row, head;
};

struct Args {
  Strided q, k, v, dout;
  void* o;      // (Tq, H, D) contiguous; read by the backward
  void* o_rest; // bf16: what the rounding of o left out, for delta; may be null
  void *dq, *dk, *dv;
  float* lse;   // (H, Tq), with lse_rest twice: see store_lse
  float* delta; // (H, Tq): dO . O; bf16: minus that, then (H, Tq) minus lse, then (H, Tq) of which every 32nd of a sequence: beyond kDeep
  const Tile* tiles;
  const void* table;  // (buckets, H) bias, or null
  const int* buckets; // (2 span + 1): bucket of distance index - span
  float* dist_part;   // (tiles, H, 2 span + 1): bias gradient by distance, or null
  int64_t tq, tk;
  int longest;  // keys of a sequence, at most
  int splits;   // of the keys among CTAs (bf16 forward)
  int heads, kv_heads, dim, span, n_buckets;
  int pack;  // heads that are neighbouring rows of a tile (bf16)
  bool causal, table_bf16, lse_rest;
  float scale;
};

__device__ __forceinline__ Seq load_tile(const Args& a, int i, int* index) {
  const int4 v = *reinterpret_cast<const int4*>(&a.tiles[i].s);
  *index = a.tiles[i].index;
  return Seq{v.x, v.y, v.z, v.w};
}

// A query that sees one key has P = 1 whatever its score: dS = 0, without the
// rounding of dP - delta.
__device__ __forceinline__ bool one_key(const Args& a, const Seq& s, int pos) { return s.lk == 1 || (a.causal && pos == 0); }

// A bias in base 2; the lowest and highest finite values stay finite.
__device__ __forceinline__ float bias_base2(float b) {
  return isinf(b) ? b : fminf(fmaxf(b * kLog2e, -CUDART_MAX_NORMAL_F), CUDART_MAX_NORMAL_F);
}

// With a bias, from this magnitude of it or of a row's maximum on, scores are taken as
// the float32 numbers that product and bias round to, and lse as two of them: next to
// a mask of 1e9 or the type's lowest value log2(sum) is less than lse's last digit, and
// P = 2^(score - lse) would not add up to 1.  Below, P loses at most 2^-12 by that.
// (Without a bias such scores have lost as much in their own rounding.)
constexpr float kDeep = 4096.f;
__device__ __forceinline__ bool deep(float x) { return fabsf(x) >= kDeep && !isinf(x); }

// lse of a row with maximum m and sum l, and what its rounding leaves out.
__device__ __forceinline__ void store_lse(const Args& a, int64_t at, float m, float l) {
  const float log = log2f(l), lse = l == 0.f ? 0.f : m + log;
  a.lse[at] = lse;
  if (a.lse_rest) a.lse[a.heads * a.tq + at] = l == 0.f ? 0.f : (m - lse) + log;
}
__device__ __forceinline__ float load_lse_rest(const Args& a, int64_t at) { return a.lse_rest ? a.lse[a.heads * a.tq + at] : 0.f; }

// Bias of one head in base 2, by clamped distance.
__device__ __forceinline__ void expand_bias_f32(const Args& a, int head, float* out, int thread, int n_threads) {
  for (int i = thread; i < 2 * a.span + 1; i += n_threads) {
    const int64_t at = (int64_t)min(max(a.buckets[i], 0), a.n_buckets - 1) * a.heads + head;
    const float b = a.table_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.table)[at])
                                 : static_cast<const float*>(a.table)[at];
    out[i] = bias_base2(b);
  }
}

// The kernels read 16 bytes at a time: what the entry points check.
inline bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}
struct Extent {
  int64_t n, stride;  // in elements
};
inline bool strides16(int size, std::initializer_list<Extent> es) {
  for (const Extent& e : es)
    if (e.n > 1 && e.stride * size % 16) return false;
  return true;
}

// attention_f32.cu, attention_fwd.cu, attention_bwd.cu
int fwd_f32(const Args& a, int n_tiles, cudaStream_t st);
int bwd_f32(const Args& a, const Tile* k_tiles, int n_q, int n_k, cudaStream_t st);
// shared memory of the bf16 forward for bias tables
constexpr int fwd_bias_bytes(int dim) { return dim <= 64 ? 12 * 1024 : 32 * 1024; }
int fwd_bf16(const Args& a, int n_tiles, cudaStream_t st);
int bwd_bf16(const Args& a, const Tile* k_tiles, int n_q, int n_k, cudaStream_t st);

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ int clamp_dist(int d, int span) { return min(max(d, -span), span) + span; }

}  // namespace attn
}  // namespace kf
