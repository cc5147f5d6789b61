// Building blocks of the bf16 attention kernels on the tensor cores: one-CTA
// tcgen05 instructions, tile loads by cp.async into the 128-byte swizzled
// layout, and the softmax arithmetic shared by forward and backward.
#pragma once

#include "attention.cuh"
#include "umma.cuh"

namespace kf {
namespace attn {

using namespace umma;

constexpr int kRows = 128;             // rows of an MMA tile, and keys or queries of a streamed tile
constexpr int kPanel = kRows * 128;    // bytes of 128 rows x 64 bf16
constexpr int kBiasPad = 160;          // distances a tile may lie past the span where it still reads the table
constexpr int kBiasBytes = 32 * 1024;  // shared memory for bias tables

template <int DP>
constexpr int tile_bytes() { return kPanel * (DP / 64); }

__host__ __device__ constexpr int bias_floats(int span) { return 2 * span + 1 + 2 * kBiasPad; }

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

// D[tmem] (+)= A[smem] B[smem]^T
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]^T: a lane holds a row of A, a column two neighbouring bf16 of it
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One arrival on `bar` when every MMA this thread has issued is complete.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
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
  constexpr int CH = DP / 8;
#pragma unroll 4
  for (int i = tid; i < kRows * CH; i += THREADS) {
    const int row = i / CH, ch = i % CH;
    const bool ok = row < n && ch * 8 < dim;
    const __nv_bfloat16* src = base;
    if (ok) {
      const int r = first_row + row;
      if (pack == 1) {
        src += (int64_t)r * row_stride + ch * 8;
      } else {
        const int tok = r / pack;
        src += (int64_t)tok * row_stride + (int64_t)(r - tok * pack) * head_stride + ch * 8;
      }
    }
    cp_async16(dst + (ch >> 3) * kPanel + sw128_offset(row, ch & 7), src, ok ? 16 : 0);
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

// The loader's side of a ring of STAGES tiles.  Item 0 was issued before and
// signals `fixed`; issue(it) starts the copies of tile it.  A thread keeps up to
// three items in flight and signals an item once its own copies have landed;
// before it blocks on a full ring it signals all it has, since the MMAs that
// free a tile may need the ones just loaded.
template <int STAGES, typename Issue>
__device__ __forceinline__ void feed_ring(int n_items, uint64_t* fixed, uint64_t* full, uint64_t* empty, volatile int* abort,
                                          Issue&& issue) {
  cp_async_commit();
  int sent = 0;  // items signalled
  auto signal = [&](int upto) {
    fence_proxy_async_smem();
    for (; sent < upto; ++sent) mbar_arrive(sent == 0 ? fixed : full + (sent - 1) % STAGES);
  };
  bool ok = true;
  for (int it = 0; it < n_items; ++it) {
    const uint32_t parity = ((it / STAGES) & 1) ^ 1;
    if (!mbar_test(empty + it % STAGES, parity)) {
      cp_async_wait<0>();
      signal(it + 1);
      if (!(ok = mbar_wait(empty + it % STAGES, parity, abort))) break;
    }
    issue(it);
    cp_async_commit();
    cp_async_wait<2>();
    if (it > 0) signal(it);  // items 0 .. it - 1 of it + 2
  }
  cp_async_wait<0>();
  if (ok) signal(n_items + 1);
}

// K-major operand (rows x DP, contraction over DP), k-step j of 16
__device__ __forceinline__ uint64_t desc_k(uint32_t tile, int j) { return smem_desc_sw128(tile + (j >> 2) * kPanel + (j & 3) * 32, 16, 1024); }
// MN-major operand (contraction over its 128 rows), k-step j of 16 rows
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile, int j) { return smem_desc_sw128(tile + j * 2048, kPanel, 1024); }

// ---- softmax arithmetic ---------------------------------------------------------

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The padded bias tables of `pack` heads: index distance + span + kBiasPad.
__device__ __forceinline__ void expand_bias_padded(const Args& a, int head0, int pack, float* out, int thread, int n_threads) {
  const int n = bias_floats(a.span);
  for (int i = thread; i < pack * n; i += n_threads) {
    const int at = min(max(i % n - kBiasPad, 0), 2 * a.span);
    const int64_t e = (int64_t)a.buckets[at] * a.heads + head0 + i / n;
    out[i] = bias_base2(a.table_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.table)[e])
                                     : static_cast<const float*>(a.table)[e]);
  }
}

}  // namespace attn
}  // namespace kf
