// Building blocks of the bf16 attention kernels on the tensor cores: one-CTA
// tcgen05 instructions, tile loads into the 128-byte swizzled layout (by TMA; the
// forward's queries, whose rows may be heads of one token, by cp.async), and the
// softmax arithmetic shared by forward and backward.
#pragma once

#include "attention.cuh"
#include "f32x2.cuh"
#include "umma.cuh"

namespace kf {
namespace attn {

using namespace umma;

constexpr int kRows = 128;             // rows of an MMA tile
constexpr int kBoxRows = 64;           // rows of a TMA box
constexpr int kBiasPad = 160;          // distances a tile may lie past the span where it still reads the table

// bytes of `rows` x DP bf16, stored as panels of 64 columns
template <int DP>
__host__ __device__ constexpr int tile_bytes(int rows) { return rows * 128 * (DP / 64); }

__host__ __device__ constexpr int bias_stride(int span) { return 2 * span + 1 + 2 * kBiasPad; }

// ---- tcgen05, one CTA --------------------------------------------------------

__device__ __forceinline__ void tmem_alloc(uint32_t* dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// The warps that issue MMAs stay converged and one elected lane issues: loop
// counters and addresses are then the warp's, in uniform registers, where the
// instruction wants them.  With a lane alone in the loop one warp issued a
// 128 x 64 x 16 product every 89 clocks, like this one every 49, which is what
// the tensor cores take.
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(is));
  return is;
}
// A value all lanes of the warp have, as one the compiler knows to be the same in all of them.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ int uniform(int v) { return __reduce_max_sync(0xffffffffu, v); }

// A shared memory operand: the descriptor's low word (address) and the high
// word, which all operands share; a step along the operand is an addition to
// the low word, so that issuing an MMA costs a few instructions.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);  // stride 1024, version 1, 128-byte swizzle

// D[tmem] (+)= A[smem] B[smem]^T, by the lane whose `leader` is set
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHi), "r"(leader)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]^T: a lane holds a row of A, a column two neighbouring bf16 of it
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHi), "r"(leader)
      : "memory");
}
// One arrival on `bar` when every MMA the leader has issued is complete.
__device__ __forceinline__ void mma_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}

// 32 columns of this thread's TMEM lane, without waiting for the data.
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// The same for 8 columns.
__device__ __forceinline__ void tmem_ld8_issue(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
// Waits for this thread's TMEM loads; the registers pass through so that no use moves above the wait.
template <int N>
__device__ __forceinline__ void tmem_wait_ld(float (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A warp's 32 rows of results, a lane to a row, on their way to memory: through
// shared memory, so that neighbouring lanes write whole lines (a lane that writes
// its row itself touches 32 lines an instruction).  The rows of a tile lie
// anywhere (heads side by side): each lane brings its row's address.
template <int DP>
__device__ __forceinline__ uint32_t staged(uint32_t stage, int row, int chunk) {
  return stage + row * (DP * 2) + ((chunk ^ (row & 7)) << 4);  // 16 bytes; both ways of access meet all banks
}
template <int DP>
__device__ __forceinline__ void stage_chunk(uint32_t stage, int chunk, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staged<DP>(stage, threadIdx.x & 31, chunk)), "r"(w0), "r"(w1), "r"(w2),
               "r"(w3)
               : "memory");
}
template <int DP>
__device__ __forceinline__ void flush_rows(uint32_t stage, __nv_bfloat16* out, bool valid, int dim) {
  constexpr int CH = DP / 8;
  __syncwarp();
  const uint32_t rows = __ballot_sync(0xffffffffu, valid);
#pragma unroll 4
  for (int k = 0; k < CH; ++k) {
    const int i = k * 32 + (threadIdx.x & 31), row = i / CH, c = i % CH;
    uint8_t* to = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), row));
    if ((rows >> row & 1) == 0 || c * 8 >= dim) continue;
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(staged<DP>(stage, row, c)) : "memory");
    *reinterpret_cast<uint4*>(to + c * 16) = v;
  }
  __syncwarp();
}

// Moves registers between the warpgroups of a CTA; the sum over its
// warpgroups must not exceed what the CTA was launched with.
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// ---- tile loads ---------------------------------------------------------------

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 128 rows x DP columns into panels of 64 columns.  Rows past n and columns past
// dim become zeros without a read: nothing outside the sequence enters an MMA.
// `pack` neighbouring rows are the heads of one token.
template <int DP, int THREADS>
__device__ __forceinline__ void load_tile_async(uint32_t dst, const __nv_bfloat16* base, int64_t row_stride, int64_t head_stride,
                                                int pack, int first_row, int n, int dim, int tid) {
  constexpr int CH = DP / 8, STEP = THREADS / CH;  // a thread's rows are STEP apart
  static_assert(STEP % 8 == 0 && kRows % STEP == 0);
  const int ch = tid % CH, row0 = tid / CH, tok = (first_row + row0) / pack;
  int head = first_row + row0 - tok * pack;
  const __nv_bfloat16* src = base + (int64_t)tok * row_stride + (int64_t)head * head_stride + ch * 8;
  const int toks = STEP / pack, heads = STEP - toks * pack;
  const int64_t step = (int64_t)toks * row_stride + (int64_t)heads * head_stride, carry = row_stride - (int64_t)pack * head_stride;
  dst += (ch >> 3) * (kRows * 128) + sw128_offset(row0, ch & 7);
  const int rows = ch * 8 < dim ? n : 0;
#pragma unroll
  for (int i = 0; i < kRows / STEP; ++i) {
    const bool ok = row0 + i * STEP < rows;
    cp_async16(dst + i * STEP * 128, ok ? src : base, ok ? 16 : 0);
    src += step, head += heads;
    if (head >= pack) head -= pack, src += carry;
  }
}

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// 3-D tiled load (column, head, row) of 64 columns x 64 rows of one head.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

__device__ __forceinline__ void st_zero16(uint32_t dst) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst), "r"(0) : "memory");
}

// One warp's loads of tiles of ROWS rows by TMA.  Rows past the sequence belong
// to its neighbour in the packed tensor: a tile that has such rows lands on a
// barrier of the warp's own and is signalled once they are overwritten by
// zeros, so that nothing outside a sequence enters an MMA.  That last step of a
// tile is left until the next tile is on its way.
template <int DP>
struct TileLoader {
  uint64_t* part;  // two barriers, count 1
  volatile int* abort;
  int used = 0;           // partial tiles so far
  bool pending = false;   // one of them is not signalled yet:
  uint32_t p_dst = 0;
  int p_rows = 0, p_n = 0;
  uint64_t* p_full = nullptr;

  __device__ __forceinline__ TileLoader(uint64_t* part_, volatile int* abort_) : part(part_), abort(abort_) {}

  __device__ __forceinline__ bool finish() {
    if (!pending) return true;
    pending = false;
    const int lane = threadIdx.x & 31;
    uint64_t* bar = part + ((used - 1) & 1);
    const uint32_t parity = ((used - 1) >> 1) & 1;
    const bool ok = mbar_wait_warp(bar, parity, abort);
    if (!ok) mbar_drain(bar, parity);
#pragma unroll
    for (int p = 0; p < DP / 64; ++p)
      for (int i = lane; i < (p_rows - p_n) * 8; i += 32) st_zero16(p_dst + p * p_rows * 128 + p_n * 128 + i * 16);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(p_full);
    return ok;
  }

  // The n (at least 1) first rows of the tile at `row` of head `head`; one arrival on `full` when it is there.
  template <int ROWS>
  __device__ __forceinline__ bool load(uint32_t dst, const CUtensorMap* map, uint64_t* full, int head, int row, int n) {
    n = min(n, ROWS);
    const bool partial = n < ROWS;
    uint64_t* bar = partial ? part + (used & 1) : full;
    if ((threadIdx.x & 31) == 0) {
      const int boxes = (n + kBoxRows - 1) / kBoxRows;
      mbar_arrive_expect_tx(bar, boxes * kBoxRows * 128 * (DP / 64));
#pragma unroll
      for (int p = 0; p < DP / 64; ++p)
        for (int b = 0; b < boxes; ++b)
          tma_load_3d(dst + p * ROWS * 128 + b * kBoxRows * 128, map, bar, p * 64, head, row + b * kBoxRows);
    }
    bool ok = true;
    if (pending) ok = finish();  // the tile before: of the other barrier, if this one is partial too
    if (partial) ++used, pending = true, p_dst = dst, p_rows = ROWS, p_n = n, p_full = full;
    return ok;
  }
};

// A ring of STAGES tiles: tile it goes to stage it % STAGES once that is free.
// load(it, stage) starts one; after an abort the loads in flight are waited for.
template <int STAGES, int DP, typename Load>
__device__ __forceinline__ void feed_ring(TileLoader<DP>& loader, int n_items, uint64_t* full, uint64_t* empty, volatile int* abort,
                                          Load&& load) {
  int it = 0;
  for (; it < n_items; ++it) {
    const uint32_t parity = ((it / STAGES) & 1) ^ 1;
    if (!__all_sync(0xffffffffu, mbar_test(empty + it % STAGES, parity))) {
      if (!loader.finish() || !mbar_wait_warp(empty + it % STAGES, parity, abort)) break;
    }
    if (!load(it, it % STAGES)) break;
  }
  loader.finish();
  if (*abort)
    for (int i = max(0, it - STAGES); i < it; ++i) mbar_drain(full + i % STAGES, (i / STAGES) & 1);
}

// Low words of operands of ROWS rows.  K-major (contraction over DP): k-step j of 16 columns.
__device__ __forceinline__ uint32_t desc_k(uint32_t tile) { return ((tile >> 4) & 0x3FFFu) | (1u << 16); }
template <int ROWS>
__host__ __device__ constexpr uint32_t step_k(int j) { return ((j >> 2) * ROWS * 128 + (j & 3) * 32) >> 4; }
// MN-major (contraction over the rows, panels of 64 columns): k-step j of 16 rows.
template <int ROWS>
__device__ __forceinline__ uint32_t desc_mn(uint32_t tile) { return ((tile >> 4) & 0x3FFFu) | ((uint32_t)(ROWS * 128 >> 4) << 16); }
__host__ __device__ constexpr uint32_t step_mn(int j) { return j * (2048 >> 4); }

// Map of a (tokens, heads, dim) bf16 tensor, boxes of 64 columns x 1 head x 64 rows.
int make_tile_map(CUtensorMap* map, const void* p, int64_t rows, int heads, int dim, int64_t row_stride, int64_t head_stride);

// ---- softmax arithmetic ---------------------------------------------------------

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The padded bias tables of `pack` heads (index distance + span + kBiasPad);
// `column` has room for the heads' columns of the learned table.  begin() starts
// the reads, so that other loads can go out before they are waited for; sync() is
// a barrier of the `n_threads` threads.
__host__ __device__ constexpr int bias_floats(int span, int n_buckets) { return bias_stride(span) + n_buckets; }

// Code that a CTA runs once costs the fetching of its instructions: the loops stay
// loops (unrolled, with the numbers in registers, the last one took 2000 clocks).
struct BiasTable {
  uint32_t raw;  // this thread's first element of the columns

  __device__ __forceinline__ uint32_t column_at(const Args& a, int head0, int i) {
    const int64_t e = (int64_t)(i % a.n_buckets) * a.heads + head0 + i / a.n_buckets;
    return a.table_bf16 ? static_cast<const uint16_t*>(a.table)[e] : static_cast<const uint32_t*>(a.table)[e];
  }
  // The bucket numbers come by cp.async, a group of their own, to where the first table will be.
  __device__ __forceinline__ void begin(const Args& a, int head0, int pack, float* out, int thread, int n_threads) {
    const int n = bias_stride(a.span);
    raw = column_at(a, head0, min(thread, pack * a.n_buckets - 1));
#pragma unroll 1
    for (int i = thread; i < n; i += n_threads)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(out + i)),
                   "l"(a.buckets + min(max(i - kBiasPad, 0), 2 * a.span))
                   : "memory");
    cp_async_commit();
  }
  // LATER: groups of cp.async since begin() that need not be complete
  template <int LATER, typename Sync>
  __device__ __forceinline__ void finish(const Args& a, int head0, int pack, float* out, float* column, int thread, int n_threads,
                                         Sync&& sync) {
    const int n = bias_stride(a.span);
#pragma unroll 1
    for (int i = thread; i < pack * a.n_buckets; i += n_threads) {
      if (i != thread) raw = column_at(a, head0, i);
      column[i] = bias_base2(__uint_as_float(a.table_bf16 ? raw << 16 : raw));
    }
    cp_async_wait<LATER>();
    sync();
#pragma unroll 1
    for (int i = thread; i < n; i += n_threads) {
      const int id = min(max(__float_as_int(out[i]), 0), a.n_buckets - 1);  // this thread's own copy
#pragma unroll 1
      for (int g = pack - 1; g >= 0; --g) out[g * n + i] = column[g * a.n_buckets + id];
    }
  }
};

// The same at once, with the bucket numbers in registers.  For dK dV, which expands
// a table inside its loop over the heads: there the rolled form costs the loop
// registers (one document of 8191 tokens: 672 us, 628 in this form).
struct BiasTableRegs {
  static constexpr int U = 8;
  uint32_t raw;  // this thread's first element of the columns
  int id[U];     // its first bucket numbers

  __device__ __forceinline__ void load(const Args& a, int i0, int n_threads) {
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = a.buckets[min(max(i0 + u * n_threads - kBiasPad, 0), 2 * a.span)];
  }
  __device__ __forceinline__ uint32_t column_at(const Args& a, int head0, int i) {
    const int64_t e = (int64_t)(i % a.n_buckets) * a.heads + head0 + i / a.n_buckets;
    return a.table_bf16 ? static_cast<const uint16_t*>(a.table)[e] : static_cast<const uint32_t*>(a.table)[e];
  }
  __device__ __forceinline__ void begin(const Args& a, int head0, int pack, int thread, int n_threads) {
    raw = column_at(a, head0, min(thread, pack * a.n_buckets - 1));
    load(a, thread, n_threads);
  }
  template <typename Sync>
  __device__ __forceinline__ void finish(const Args& a, int head0, int pack, float* out, float* column, int thread, int n_threads,
                                         Sync&& sync) {
    const int n = bias_stride(a.span);
    for (int i = thread; i < pack * a.n_buckets; i += n_threads) {
      if (i != thread) raw = column_at(a, head0, i);
      column[i] = bias_base2(__uint_as_float(a.table_bf16 ? raw << 16 : raw));
    }
    sync();
    for (int i0 = thread; i0 < n; i0 += U * n_threads) {
      if (i0 != thread) load(a, i0, n_threads);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * n_threads;
        if (i >= n) break;
        for (int g = 0; g < pack; ++g) out[g * n + i] = column[g * a.n_buckets + min(max(id[u], 0), a.n_buckets - 1)];
      }
    }
  }
};

template <typename Sync>
__device__ __forceinline__ void expand_bias(const Args& a, int head0, int pack, float* out, float* column, int thread, int n_threads,
                                            Sync&& sync) {
  BiasTableRegs t;
  t.begin(a, head0, pack, thread, n_threads);
  t.finish(a, head0, pack, out, column, thread, n_threads, sync);
}

}  // namespace attn
}  // namespace kf
