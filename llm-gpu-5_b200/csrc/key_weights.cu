// Accumulated attention weights of a prompt: for every key j of a key head,
//   w[j] = sum over the head's query heads and the queries i >= max(j, first_query), i < length, of
//          p_ij = exp(scale q_i . k_j - lse_i),
// the column sums of the causal softmax whose row statistics attn_fwd left in lse.  The T x T matrix
// (attn_probs, the reference's cache_attn_weights) is never stored.
//
// A thread takes one key and a CTA 128 of them; queries pass through shared memory in tiles of 32 and
// a thread forms 8 scores at a time, so that each value of its key is read once for 8 products.
#include "kv4.cuh"
#include "tc_common.cuh"
#include <math.h>

namespace attn {

constexpr int KW_KEYS = 128;
constexpr int KW_QUERIES = 32;

struct KeyWeights {
  const void *q, *k;
  const float *lse, *w_in;
  float* w_out;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, w_sb, w_sh;
  int NH, NKV, G, T, D, first;
  const int* lengths;
  float scale_log2;
};

__device__ __forceinline__ float tf32_cut(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }

template <typename T, bool TF32>
__global__ void __launch_bounds__(KW_KEYS) key_weights_simt_kernel(const KeyWeights p) {
  extern __shared__ float sm[];
  float* sk = sm;                       // [D][KW_KEYS]
  float* sq = sk + p.D * KW_KEYS;       // [KW_QUERIES][D]
  float* sl = sq + KW_QUERIES * p.D;    // [KW_QUERIES]
  grid_dependency_wait();
  grid_dependents_launch();
  const int ntile = (p.T + KW_KEYS - 1) / KW_KEYS;
  const int bh = blockIdx.x / ntile, j0 = (blockIdx.x % ntile) * KW_KEYS;
  const int b = bh / p.NKV, kvh = bh % p.NKV;
  const int n = seq_length(p.lengths, b, p.T);
  const int j = j0 + threadIdx.x;
  const T* kb = (const T*)p.k + b * p.k_sb + kvh * p.k_sh;
  for (int i = threadIdx.x; i < KW_KEYS * p.D; i += KW_KEYS) {
    const int r = i / p.D, d = i - r * p.D;
    float x = j0 + r < n ? Elem<T>::load(kb + (int64_t)(j0 + r) * p.k_st + d) : 0.f;
    sk[d * KW_KEYS + r] = TF32 ? tf32_cut(x) : x;
  }
  float total = 0.f;
  for (int g = 0; g < p.G; ++g) {
    const int h = kvh * p.G + g;
    const T* qb = (const T*)p.q + b * p.q_sb + h * p.q_sh;
    const float* lse = p.lse + ((int64_t)b * p.NH + h) * p.T;
    for (int i0 = max(j0, p.first); i0 < n; i0 += KW_QUERIES) {
      __syncthreads();
      for (int e = threadIdx.x; e < KW_QUERIES * p.D; e += KW_KEYS) {
        const int r = e / p.D, d = e - r * p.D;
        float x = i0 + r < n ? Elem<T>::load(qb + (int64_t)(i0 + r) * p.q_st + d) : 0.f;
        sq[e] = TF32 ? tf32_cut(x) : x;
      }
      if (threadIdx.x < KW_QUERIES) sl[threadIdx.x] = i0 + threadIdx.x < n ? lse[i0 + threadIdx.x] * 1.4426950408889634f : 0.f;
      __syncthreads();
      for (int r0 = 0; r0 < KW_QUERIES; r0 += 8) {
        float acc[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) acc[r] = 0.f;
        for (int d = 0; d < p.D; ++d) {
          const float x = sk[d * KW_KEYS + threadIdx.x];
#pragma unroll
          for (int r = 0; r < 8; ++r) acc[r] += x * sq[(r0 + r) * p.D + d];
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int i = i0 + r0 + r;
          if (i < n && i >= j) total += exp2f(fmaf(acc[r], p.scale_log2, -sl[r0 + r]));
        }
      }
    }
  }
  if (j < p.T) {
    const int64_t at = b * p.w_sb + kvh * p.w_sh + j;
    p.w_out[at] = (p.w_in ? p.w_in[at] : 0.f) + (j < n ? total : 0.f);
  }
}

static int key_weights_simt(const KeyWeights& p, int B, int dtype, cudaStream_t s) {
  const size_t smem = ((size_t)p.D * (KW_KEYS + KW_QUERIES) + KW_QUERIES) * sizeof(float);
  const int64_t grid = (int64_t)B * p.NKV * ((p.T + KW_KEYS - 1) / KW_KEYS);
  auto kern = dtype == ATTN_BF16 ? key_weights_simt_kernel<__nv_bfloat16, false>
              : dtype == ATTN_TF32 ? key_weights_simt_kernel<float, true> : key_weights_simt_kernel<float, false>;
  ATTN_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const cudaError_t e = launch_pdl(kern, dim3((unsigned)grid), dim3(KW_KEYS), smem, s, p);
  count_launch();
  return check_launch("key_weights_simt_kernel", e);
}

}  // namespace attn

using namespace attn;

extern "C" int attn_key_weights(const void* q, const void* k, const float* lse, const float* weights_in,
                                float* weights_out, int B, int NH, int NKV, int T, int D, int64_t q_sb, int64_t q_st,
                                int64_t q_sh, int64_t k_sb, int64_t k_st, int64_t k_sh, int64_t w_sb, int64_t w_sh,
                                int first_query, const int* lengths, float scale, int dtype, void* stream) {
  clear_error();
  ATTN_REQUIRE(q && k && lse && weights_out, "attn_key_weights: null pointer argument");
  ATTN_REQUIRE(dtype == ATTN_F32 || dtype == ATTN_BF16 || dtype == ATTN_TF32, "attn_key_weights: bad dtype");
  ATTN_REQUIRE(B > 0 && NH > 0 && NKV > 0 && T > 0 && D > 0, "attn_key_weights: sizes must be positive");
  ATTN_REQUIRE(NH % NKV == 0, "attn_key_weights: %d query heads are no multiple of %d key heads", NH, NKV);
  ATTN_REQUIRE(first_query >= 0, "attn_key_weights: first_query must not be negative");
  ATTN_REQUIRE(q_sb >= 0 && q_st >= 0 && q_sh >= 0 && k_sb >= 0 && k_st >= 0 && k_sh >= 0 && w_sb >= 0 && w_sh >= 0,
               "attn_key_weights: strides must not be negative");
  const size_t esz = dtype == ATTN_BF16 ? 2 : 4;
  ATTN_REQUIRE(aligned(q, esz) && aligned(k, esz) && aligned(lse, 4), "attn_key_weights: misaligned tensor");
  if (D > 128) {
    set_error("attn_key_weights: head_dim %d not supported (up to 128)", D);
    return ATTN_ERR_UNSUPPORTED;
  }
  if ((int64_t)B * NKV * ((T + KW_KEYS - 1) / KW_KEYS) >= (int64_t)1 << 31) {
    set_error("attn_key_weights: too many key tiles for one launch; split the batch into several calls");
    return ATTN_ERR_UNSUPPORTED;
  }
  const KeyWeights p = {q, k, lse, weights_in, weights_out, q_sb, q_st, q_sh, k_sb, k_st, k_sh, w_sb, w_sh,
                        NH, NKV, NH / NKV, T, D, first_query, lengths, scale * 1.4426950408889634f};
  return key_weights_simt(p, B, dtype, as_stream(stream));
}
