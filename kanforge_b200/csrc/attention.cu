// C ABI of packed attention: checks, tiling and dispatch by type, and the
// last step of the bias gradient.
#include "attention_tc.cuh"

namespace kf {
namespace {

using namespace attn;

constexpr int kWorkspaceRows = 3;  // of (H, Tq) floats at Args::delta

// The bias gradient by distance: the tiles' sums of one (head, distance), 32
// distances by 8 slices of the tiles, joined in order.
__global__ void __launch_bounds__(256) attention_dist(const float* part, int n_tiles, int heads, int n_dist, float* out) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, e = blockIdx.x * 32 + lane, head = blockIdx.y;
  float v = 0.f;
  if (e < n_dist) {
#pragma unroll 8
    for (int t = slice; t < n_tiles; t += 8) v += part[((int64_t)t * heads + head) * n_dist + e];
  }
  s[slice][lane] = v;
  __syncthreads();
  if (slice != 0 || e >= n_dist) return;
  for (int i = 1; i < 8; ++i) v += s[i][lane];
  out[(int64_t)head * n_dist + e] = v;
}

// ... and by bucket: a warp per (bucket, head), lanes over the distances.
__global__ void __launch_bounds__(256) attention_dtable(const float* dist, const int* buckets, int n_dist, int heads, int n_buckets,
                                                        void* out, bool bf16) {
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= heads * n_buckets) return;
  const int bucket = i / heads, head = i - bucket * heads;
  float v = 0.f;
#pragma unroll 4
  for (int e = lane; e < n_dist; e += 32) v += buckets[e] == bucket ? dist[(int64_t)head * n_dist + e] : 0.f;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  if (lane != 0) return;
  if (bf16)
    static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(out)[i] = v;
}

int check_attention(const char* fn, const kf_attention_desc* d) {
  KF_CHECK_ARG(d != nullptr, "%s: null descriptor", fn);
  KF_CHECK_ARG(d->heads >= 1 && d->kv_heads >= 1 && d->heads % d->kv_heads == 0, "%s: %d heads do not divide over %d key heads", fn,
               d->heads, d->kv_heads);
  KF_CHECK_ARG(d->heads <= 65535, "%s: %d heads", fn, d->heads);
  KF_CHECK_ARG(d->dim >= 8 && d->dim <= kMaxDim && d->dim % 8 == 0, "%s: head width %d is not a multiple of 8 up to %d", fn, d->dim,
               kMaxDim);
  KF_CHECK_ARG(d->dtype == KF_DTYPE_F32 || d->dtype == KF_DTYPE_BF16, "%s: types must be float32 or bfloat16", fn);
  KF_CHECK_ARG(d->tq >= 0 && d->tk >= 0 && d->longest >= 0, "%s: negative size", fn);
  KF_CHECK_ARG(d->span >= 0 && d->span <= kMaxSpan, "%s: bias distances up to %d are outside [0, %d]", fn, d->span, kMaxSpan);
  KF_CHECK_ARG(d->n_buckets >= 0 && d->n_buckets <= kMaxBuckets, "%s: %d buckets exceed %d", fn, d->n_buckets, kMaxBuckets);
  return KF_OK;
}

// Rows of a tile of the forward's queries (pass 0), the backward's queries (1)
// and its keys (2), and how many neighbouring rows are heads of one token.
// bf16 packs the heads that share a key head, unless their bias tables would
// not fit in shared memory (with D <= 64: twice an SM).  Few queries then fill a
// tile: 32 x 16 queries of 32 heads of 128 on 8 key heads over 4096 keys take 120 us,
// unpacked 353; 16 documents of up to 2000 tokens, 12 heads of 64 on 4: 85 and 91 us;
// one of 8191, 16 heads of 128 on 4: 238 and 241 us.
void tiling(const kf_attention_desc* d, int pass, int32_t* rows, int32_t* pack) {
  *pack = 1;
  *rows = d->dtype == KF_DTYPE_F32 ? 64 : pass == 0 && d->dim > 64 ? 256 : 128;
  if (d->dtype == KF_DTYPE_F32 || pass > 0) return;
  const int group = d->heads / d->kv_heads;
  if (d->n_buckets == 0 || group * bias_floats(d->span, d->n_buckets) * (int)sizeof(float) <= fwd_bias_bytes(d->dim)) *pack = group;
}

bool rows_aligned(const kf_attention_desc* d, std::initializer_list<const void*> ps) {
  return aligned16(ps) && strides16(d->dtype == KF_DTYPE_F32 ? 4 : 2, {{d->tq, d->q_row}, {d->heads, d->q_head}, {d->tk, d->k_row},
                                                                       {d->kv_heads, d->k_head}, {d->tk, d->v_row}, {d->kv_heads, d->v_head}});
}

Args make_args(const kf_attention_desc* d) {
  Args a{};
  a.heads = d->heads, a.kv_heads = d->kv_heads, a.dim = d->dim, a.span = d->span, a.n_buckets = d->n_buckets;
  a.causal = d->causal != 0, a.table_bf16 = d->table_dtype == KF_DTYPE_BF16;
  a.lse_rest = d->lse_rest != 0, a.scale = d->scale, a.tq = d->tq, a.tk = d->tk, a.longest = d->longest;
  a.q = {nullptr, d->q_row, d->q_head};
  a.k = {nullptr, d->k_row, d->k_head};
  a.v = {nullptr, d->v_row, d->v_head};
  a.dout = {nullptr, (int64_t)d->heads * d->dim, d->dim};
  return a;
}

}  // namespace
}  // namespace kf

int kf::attn::make_tile_map(CUtensorMap* map, const void* p, int64_t rows, int heads, int dim, int64_t row_stride,
                            int64_t head_stride) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn) : nullptr;
  }();
  if (encode == nullptr) {
    set_error("cuTensorMapEncodeTiled is not available from the driver");
    return KF_ERR_CUDA;
  }
  // the stride of a dimension of size one is never used, but it is checked
  const cuuint64_t pitch = (cuuint64_t)(dim + 7) / 8 * 16;
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  cuuint64_t strides[2] = {heads > 1 ? (cuuint64_t)head_stride * 2 : pitch, rows > 1 ? (cuuint64_t)row_stride * 2 : pitch};
  cuuint32_t box[3] = {64, 1, (cuuint32_t)kBoxRows}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  KF_CHECK_ARG(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (%d) for %lld rows x %d heads x %d, strides %lld and %lld", (int)r,
               (long long)rows, heads, dim, (long long)row_stride, (long long)head_stride);
  return KF_OK;
}

extern "C" int kf_attention_tiling(const kf_attention_desc* d, int pass, int32_t* rows, int32_t* pack) {
  using namespace kf;
  clear_error();
  if (int rc = check_attention("kf_attention_tiling", d)) return rc;
  KF_CHECK_ARG(pass >= 0 && pass <= 2 && rows && pack, "kf_attention_tiling: bad argument");
  tiling(d, pass, rows, pack);
  return KF_OK;
}

extern "C" int kf_attention_fwd(const void* q, const void* k, const void* v, const int32_t* q_tiles, int32_t n_q_tiles, const void* table, const int32_t* buckets, void* o, void* o_rest,
                                float* lse, const kf_attention_desc* d, void* stream) {
  using namespace kf;
  clear_error();
  if (int rc = check_attention("kf_attention_fwd", d)) return rc;
  if (n_q_tiles == 0) return KF_OK;
  KF_CHECK_ARG(n_q_tiles > 0 && (int64_t)n_q_tiles * d->heads < (1ll << 31), "kf_attention_fwd: bad tile count");
  KF_CHECK_ARG(q && o && q_tiles && (d->tk == 0 || (k && v)), "kf_attention_fwd: null argument");
  KF_CHECK_ARG((table == nullptr) == (buckets == nullptr) && (table == nullptr || d->n_buckets > 0), "kf_attention_fwd: the bias needs a table and buckets");
  KF_CHECK_ARG(rows_aligned(d, {q, k, v, o, o_rest, q_tiles}), "kf_attention_fwd: rows must start at multiples of 16 bytes");
  if (int rc = bind_device(q)) return rc;
  Args a = make_args(d);
  a.q.p = q, a.k.p = k, a.v.p = v, a.o = o, a.o_rest = o_rest, a.lse = lse, a.table = table, a.buckets = buckets;
  a.tiles = reinterpret_cast<const Tile*>(q_tiles);
  int rows;
  tiling(d, 0, &rows, &a.pack);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return d->dtype == KF_DTYPE_BF16 ? fwd_bf16(a, n_q_tiles, st) : fwd_f32(a, n_q_tiles, st);
}

extern "C" int64_t kf_attention_bwd_workspace(int32_t n_q_tiles, const kf_attention_desc* d) {
  if (d == nullptr || n_q_tiles < 0) return 0;
  return kf::kWorkspaceRows * (int64_t)d->heads * d->tq + (d->n_buckets > 0 ? ((int64_t)n_q_tiles + 1) * d->heads * (2 * d->span + 1) : 0);
}

extern "C" int kf_attention_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_rest, const void* dout, const float* lse,
                                const int32_t* q_tiles, int32_t n_q_tiles, const int32_t* k_tiles,
                                int32_t n_k_tiles, const void* table, const int32_t* buckets, void* dq, void* dk, void* dv,
                                void* dtable, float* workspace, const kf_attention_desc* d, void* stream) {
  using namespace kf;
  clear_error();
  if (int rc = check_attention("kf_attention_bwd", d)) return rc;
  KF_CHECK_ARG(n_q_tiles >= 0 && n_k_tiles >= 0 && (int64_t)std::max(n_q_tiles, n_k_tiles) * d->heads < (1ll << 31),
               "kf_attention_bwd: bad tile count");
  const bool any = n_q_tiles > 0 || n_k_tiles > 0;  // each pass reads the rows of both sides
  KF_CHECK_ARG(!any || d->tq == 0 || (q && o && dout && lse && workspace), "kf_attention_bwd: null argument");
  KF_CHECK_ARG(!any || d->tk == 0 || (k && v), "kf_attention_bwd: null argument");
  KF_CHECK_ARG(n_q_tiles == 0 || (d->tq > 0 && dq && q_tiles), "kf_attention_bwd: null argument");
  KF_CHECK_ARG(n_k_tiles == 0 || (d->tk > 0 && dk && dv && k_tiles), "kf_attention_bwd: null argument");
  KF_CHECK_ARG((table == nullptr) == (buckets == nullptr) && (table == nullptr || d->n_buckets > 0), "kf_attention_bwd: the bias needs a table and buckets");
  KF_CHECK_ARG(dtable == nullptr || (table != nullptr && workspace != nullptr), "kf_attention_bwd: dtable needs a table and workspace");
  KF_CHECK_ARG(!any || d->tq == 0 || d->dtype == KF_DTYPE_F32 || o_rest != nullptr, "kf_attention_bwd: bf16 needs o_rest");
  KF_CHECK_ARG(rows_aligned(d, {q, k, v, o, o_rest, dout, dq, dk, dv, q_tiles, k_tiles}),
               "kf_attention_bwd: rows must start at multiples of 16 bytes");
  if (n_q_tiles == 0 && n_k_tiles == 0 && dtable == nullptr) return KF_OK;
  if (int rc = bind_device(n_q_tiles ? q : n_k_tiles ? k : dtable)) return rc;
  Args a = make_args(d);
  a.q.p = q, a.k.p = k, a.v.p = v, a.dout.p = dout, a.o = const_cast<void*>(o), a.o_rest = const_cast<void*>(o_rest), a.lse = const_cast<float*>(lse);
  a.dq = dq, a.dk = dk, a.dv = dv, a.table = table, a.buckets = buckets;
  a.tiles = reinterpret_cast<const Tile*>(q_tiles);
  a.delta = workspace;
  float* dist = workspace + kWorkspaceRows * (int64_t)d->heads * d->tq;  // (H, 2 span + 1), then the tiles' parts
  const int n_dist = 2 * d->span + 1;
  a.dist_part = dtable != nullptr ? dist + (int64_t)d->heads * n_dist : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Tile* kt = reinterpret_cast<const Tile*>(k_tiles);
  int rows;
  tiling(d, 1, &rows, &a.pack);
  int rc = d->dtype == KF_DTYPE_BF16 ? bwd_bf16(a, kt, n_q_tiles, n_k_tiles, st) : bwd_f32(a, kt, n_q_tiles, n_k_tiles, st);
  if (rc || dtable == nullptr) return rc;
  attention_dist<<<dim3((unsigned)cdiv(n_dist, 32), d->heads), 256, 0, st>>>(a.dist_part, n_q_tiles, d->heads, n_dist, dist);
  attention_dtable<<<(unsigned)cdiv(d->heads * d->n_buckets, 8), 256, 0, st>>>(dist, buckets, n_dist, d->heads, d->n_buckets, dtable,
                                                                               a.table_bf16);
  return check_launch("kf_attention_bwd");
}
