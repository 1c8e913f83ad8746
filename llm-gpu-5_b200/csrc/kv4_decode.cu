// Single-query decode attention over the 4-bit cache, with the attention weights accumulated per key.
//
// For every query head h of sequence b, with n = lengths[b] cached rows of its key head,
//   s_j = scale * q . k_j,  lse = log sum_j exp(s_j),  p_j = exp(s_j - lse),  o = sum_j p_j v_j,
// and weights_out[j] = weights_in[j] + sum over the key head's query heads of p_j.  No rows: o = 0,
// lse = -inf, no weight.  In a group, k = n s + m, so q . k_j = s sum_d q_d n_d + m sum_d q_d, and the
// codes enter the products as small integers.  All sums and softmax statistics are float32.
//
// The length is split over CTAs; each writes an unnormalised partial state (m, l, o[D]) and, where
// weights are wanted, its p relative to its own maximum; the combine kernel merges the states and adds
// the weights.
#include "kv4.cuh"
#include <math.h>

namespace attn {

constexpr int KD_THREADS = 128;
constexpr int KD_CHUNK = 256;    // keys per split
constexpr int KD_WCHUNK = 1024;  // keys per combine CTA

struct Kv4Decode {
  const void* q;
  void* o;
  float* lse;
  const int* lengths;
  const float* w_in;
  float* w_out;
  int64_t q_sb, q_sh, o_sb, o_sh, w_sb, w_sh;
  int NH, NKV, G, L, ns;
  float scale_log2;
  float* states;  // [B*NH][ns][D + 2]: max (log2 units), sum, unnormalised o
  float* probs;   // [B*NH][L]: 2^(s - the split's max); NULL without weights
};

static int kd_splits(int L) { return (L + KD_CHUNK - 1) / KD_CHUNK; }
static size_t kd_states(int64_t BH, int L, int D) { return ((size_t)BH * kd_splits(L) * (D + 2) + 3) / 4 * 4; }

__device__ __forceinline__ float block_reduce(float v, float* red, bool is_max) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, off);
    v = is_max ? fmaxf(v, u) : v + u;
  }
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < KD_THREADS / 32; ++i) v = is_max ? fmaxf(v, red[i]) : v + red[i];
  return v;
}

template <typename T, int D>
__global__ void __launch_bounds__(KD_THREADS) kv4_decode_partial_kernel(const Kv4View c, const Kv4Decode p) {
  constexpr int G = kv4_groups(D), GS = kv4_group(D);
  __shared__ float sq[D], sp[KD_CHUNK], red[KD_THREADS / 32];
  grid_dependency_wait();
  grid_dependents_launch();
  const int bh = blockIdx.x / p.ns, split = blockIdx.x % p.ns;
  const int b = bh / p.NH, h = bh % p.NH, kvh = h / p.G;
  const int n = seq_length(p.lengths, b, p.L);
  const int l0 = split * KD_CHUNK, l1 = min(n, l0 + KD_CHUNK);
  const T* q = (const T*)p.q + b * p.q_sb + h * p.q_sh;
  for (int d = threadIdx.x; d < D; d += KD_THREADS) sq[d] = Elem<T>::load(q + d) * p.scale_log2;
  __syncthreads();
  const int64_t row0 = b * c.sb + kvh * c.sh;
  float mx = -INFINITY;
  for (int j = l0 + threadIdx.x; j < l1; j += KD_THREADS) {
    const uint8_t* code = c.codes + (row0 + j) * (D / 2);
    float s = 0.f;
    for (int g = 0; g < G; ++g) {
      float dot = 0.f, qs = 0.f;
      for (int d = 0; d < GS; ++d) {
        const float x = sq[g * GS + d];
        dot += x * (float)((code[(g * GS + d) / 2] >> (4 * (d & 1))) & 15);
        qs += x;
      }
      const float2 sm = __half22float2(c.params[(row0 + j) * G + g]);
      s += sm.x * dot + sm.y * qs;
    }
    sp[j - l0] = s;
    mx = fmaxf(mx, s);
  }
  mx = block_reduce(mx, red, true);
  float sum = 0.f;
  for (int j = l0 + threadIdx.x; j < l1; j += KD_THREADS) {
    const float e = exp2f(sp[j - l0] - mx);
    sp[j - l0] = e;
    sum += e;
    if (p.probs) p.probs[(int64_t)bh * p.L + j] = e;
  }
  sum = block_reduce(sum, red, false);
  __syncthreads();
  float* st = p.states + ((int64_t)bh * p.ns + split) * (D + 2);
  for (int d = threadIdx.x; d < D; d += KD_THREADS) {
    float acc = 0.f;
    for (int j = l0; j < l1; ++j) {
      const int64_t row = c.si + row0 + j;
      const float2 sm = __half22float2(c.params[row * G + d / GS]);
      acc += sp[j - l0] * fmaf((float)((c.codes[row * (D / 2) + d / 2] >> (4 * (d & 1))) & 15), sm.x, sm.y);
    }
    st[2 + d] = acc;
  }
  if (threadIdx.x == 0) {
    st[0] = mx;
    st[1] = sum;
  }
}

// One CTA per (KD_WCHUNK keys, sequence, key head); the first of them also writes o and lse.
template <typename T, int D>
__global__ void __launch_bounds__(KD_THREADS) kv4_decode_combine_kernel(const Kv4Decode p) {
  __shared__ float red[KD_THREADS / 32];
  grid_dependency_wait();
  grid_dependents_launch();
  const int wchunks = p.probs ? (p.L + KD_WCHUNK - 1) / KD_WCHUNK : 1;
  const int bk = blockIdx.x / wchunks, chunk = blockIdx.x % wchunks;
  const int b = bk / p.NKV, kvh = bk % p.NKV;
  const int n = seq_length(p.lengths, b, p.L);
  const int j0 = chunk * KD_WCHUNK, j1 = min(p.L, j0 + KD_WCHUNK);
  constexpr int PER = KD_WCHUNK / KD_THREADS;
  float w[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) w[i] = 0.f;
  for (int g = 0; g < p.G; ++g) {
    const int h = kvh * p.G + g, bh = b * p.NH + h;
    const float* st = p.states + (int64_t)bh * p.ns * (D + 2);
    float mx = -INFINITY, sum = 0.f;
    for (int i = threadIdx.x; i < p.ns; i += KD_THREADS) mx = fmaxf(mx, st[(int64_t)i * (D + 2)]);
    mx = block_reduce(mx, red, true);
    if (mx == -INFINITY) mx = 0.f;
    for (int i = threadIdx.x; i < p.ns; i += KD_THREADS)
      sum += st[(int64_t)i * (D + 2) + 1] * exp2f(st[(int64_t)i * (D + 2)] - mx);
    sum = block_reduce(sum, red, false);
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    if (chunk == 0) {
      for (int d = threadIdx.x; d < D; d += KD_THREADS) {
        float acc = 0.f;
        for (int i = 0; i < p.ns; ++i) acc += st[(int64_t)i * (D + 2) + 2 + d] * exp2f(st[(int64_t)i * (D + 2)] - mx);
        Elem<T>::store((T*)p.o + b * p.o_sb + h * p.o_sh + d, acc * inv);
      }
      if (threadIdx.x == 0 && p.lse) p.lse[bh] = n > 0 ? (mx + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
    if (p.probs) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int j = j0 + i * KD_THREADS + threadIdx.x;
        if (j < j1 && j < n)
          w[i] += p.probs[(int64_t)bh * p.L + j] * exp2f(st[(int64_t)(j / KD_CHUNK) * (D + 2)] - mx) * inv;
      }
    }
  }
  if (p.probs) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = j0 + i * KD_THREADS + threadIdx.x;
      if (j < j1) {
        const int64_t at = b * p.w_sb + kvh * p.w_sh + j;
        p.w_out[at] = (p.w_in ? p.w_in[at] : 0.f) + w[i];
      }
    }
  }
}

template <typename T, int D>
static int kv4_decode_d(const Kv4View& c, const Kv4Decode& p, int B, cudaStream_t s) {
  cudaError_t e = launch_pdl(kv4_decode_partial_kernel<T, D>, dim3((unsigned)p.ns * B * p.NH), dim3(KD_THREADS), 0, s, c, p);
  count_launch();
  if (int rc = check_launch("kv4_decode_partial_kernel", e)) return rc;
  const int wc = p.probs ? (p.L + KD_WCHUNK - 1) / KD_WCHUNK : 1;
  e = launch_pdl(kv4_decode_combine_kernel<T, D>, dim3((unsigned)wc * B * p.NKV), dim3(KD_THREADS), 0, s, p);
  count_launch();
  return check_launch("kv4_decode_combine_kernel", e);
}

template <typename T>
static int kv4_decode_t(const Kv4View& c, const Kv4Decode& p, int B, int D, cudaStream_t s) {
  switch (D) {
    case 16: return kv4_decode_d<T, 16>(c, p, B, s);
    case 32: return kv4_decode_d<T, 32>(c, p, B, s);
    case 64: return kv4_decode_d<T, 64>(c, p, B, s);
    case 128: return kv4_decode_d<T, 128>(c, p, B, s);
  }
  return ATTN_ERR_UNSUPPORTED;
}

}  // namespace attn

using namespace attn;

extern "C" size_t attn_kv4_decode_workspace_size(int B, int NH, int L, int D, int weights) {
  if (B <= 0 || NH <= 0 || L <= 0 || D <= 0) return 0;
  return (kd_states((int64_t)B * NH, L, D) + (weights ? (size_t)B * NH * L : 0)) * sizeof(float);
}

extern "C" int attn_kv4_decode(const void* q, const void* codes, const void* params, void* o, float* lse, int B, int NH,
                               int NKV, int L, int D, int64_t q_sb, int64_t q_sh, int64_t o_sb, int64_t o_sh,
                               int64_t c_si, int64_t c_sb, int64_t c_sh, int capacity, const int* lengths,
                               const float* weights_in, float* weights_out, int64_t w_sb, int64_t w_sh, float scale,
                               int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  ATTN_REQUIRE(q && o, "attn_kv4_decode: null pointer argument");
  ATTN_REQUIRE(dtype == ATTN_F32 || dtype == ATTN_BF16, "attn_kv4_decode: dtype must be ATTN_F32 or ATTN_BF16");
  ATTN_REQUIRE(NH > 0 && NKV > 0 && NH % NKV == 0, "attn_kv4_decode: %d query heads are no multiple of %d cached heads", NH, NKV);
  const Kv4View c = {(uint8_t*)codes, (__half2*)params, c_si, c_sb, c_sh, capacity};
  if (int rc = kv4_check("attn_kv4_decode", c, B, NKV, D)) return rc;
  ATTN_REQUIRE(L > 0 && L <= capacity, "attn_kv4_decode: length %d outside 1 .. capacity %d", L, capacity);
  ATTN_REQUIRE(q_sb >= 0 && q_sh >= 0 && o_sb >= 0 && o_sh >= 0 && w_sb >= 0 && w_sh >= 0, "attn_kv4_decode: strides must not be negative");
  ATTN_REQUIRE(!weights_in || weights_out, "attn_kv4_decode: weights_in needs weights_out");
  if ((int64_t)B * NH * kd_splits(L) >= (int64_t)1 << 31) {
    set_error("attn_kv4_decode: B*NH*L is too large for one launch; split the batch into several calls");
    return ATTN_ERR_UNSUPPORTED;
  }
  const size_t need = attn_kv4_decode_workspace_size(B, NH, L, D, weights_out != nullptr);
  if (!workspace || workspace_bytes < need) {
    set_error("attn_kv4_decode: workspace of %zu bytes required", need);
    return ATTN_ERR_WORKSPACE;
  }
  ATTN_REQUIRE(aligned(workspace, 16), "attn_kv4_decode: workspace must be 16-byte aligned");
  Kv4Decode p = {};
  p.q = q; p.o = o; p.lse = lse; p.lengths = lengths; p.w_in = weights_in; p.w_out = weights_out;
  p.q_sb = q_sb; p.q_sh = q_sh; p.o_sb = o_sb; p.o_sh = o_sh; p.w_sb = w_sb; p.w_sh = w_sh;
  p.NH = NH; p.NKV = NKV; p.G = NH / NKV; p.L = L; p.ns = kd_splits(L);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.states = (float*)workspace;
  p.probs = weights_out ? p.states + kd_states((int64_t)B * NH, L, D) : nullptr;
  return dtype == ATTN_BF16 ? kv4_decode_t<__nv_bfloat16>(c, p, B, D, as_stream(stream)) : kv4_decode_t<float>(c, p, B, D, as_stream(stream));
}
