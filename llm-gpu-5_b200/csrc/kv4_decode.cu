// Single-query decode attention over the 4-bit cache, with the attention weights accumulated per key.
//
// For every query head h of sequence b, with n = lengths[b] cached rows of its key head,
//   s_j = scale * q . k_j,  lse = log sum_j exp(s_j),  p_j = exp(s_j - lse),  o = sum_j p_j v_j,
// and weights_out[j] = weights_in[j] + sum over the key head's query heads of p_j.  No rows: o = 0,
// lse = -inf, no weight.  In a group k = n s + m, so
//   q . k_j = s_j sum_d q_d n_jd + m_j sum_d q_d          (the first sum a product with small integers)
//   o_d     = sum_j (p_j s_j) n_jd + sum_j p_j m_j        (likewise; the second sum has no d)
// A row of 64 values is 36 bytes, so at the HBM rate an SM receives a key and its value every 3 cycles: too
// fast for 128 multiply-adds and as many conversions on the CUDA cores.  Both integer products go to
// mma.sync (m16n8k16, f16 operands, f32 accumulation; a matrix with one useful column of eight for a
// single query, which the idle tensor pipe does not mind), with the codes as the A operand:
//   - n as a float16 costs no conversion: its four bits in the mantissa of a float16 with a zero exponent
//     are a subnormal number, exactly n times a power of two.  The tensor core aligns products by their
//     operands' exponents, -14 for any subnormal, and drops what lies 24 bits below the largest: codes at
//     the top of the mantissa (n * 2^-18) keep float32's accuracy, for a shift and an AND per pair; codes in the
//     second nibble (n * 2^-20) keep 2^-22 and save half the shifts; codes left where they are (n * 2^-24, or
//     16 n * 2^-24 in the second nibble) save them all and keep 2^-17.  float32 calls use the first, the scores
//     of bfloat16 ones the second, and their value product (the output keeps 2^-9) the third.
//   - which element sits in which k slot does not matter as long as the query agrees, so a lane takes
//     consecutive codes of a key's row.
//   - q is scaled by a power of two to below 2^12: bfloat16 elements are exact down to 2^-28 of the row's largest,
//     smaller ones off by at most 2^-36 of it.  float32 ones go as two float16 parts in two columns of the same
//     product (good to 2^-22 of themselves or 2^-36 of the largest).
//   - p s is formed with p relative to a reference, in place of the scores' maximum, that keeps the largest p s of a
//     query and group between 2^7 and 2^15 (float32 outputs: 2 and 2^15).  So what a row's scale costs the others in
//     digits follows from p s, their shares of the output: each keeps 11 bits down to 2^-22 of the largest, and is off
//     by at most 2^-32 of it below.  For float32 outputs p s goes as two parts, the second 2^11 times too large so that
//     small ones keep it too: 22 bits down to 2^-16 of the largest, 2^-37 of it below.
//
// A warp takes tiles of 64 keys (32 at head_dim 128) through a ring of its own of cp.async stages (no barrier
// between warps): scores into shared memory, then one key per lane for the softmax, whose reference moves only
// when a p s passes 2^15 (the accumulators are rescaled then; a vote per tile finds that out, cheaper than every
// query's maximum), then p s back as the B operand.  The length is split over the CTAs of a cluster, up to eight,
// which merge their states (m, l, o[D]) through distributed shared memory and add the weights of their own keys: one
// launch, up to about as many CTAs as the GPU holds at once.  Otherwise (many heads, or few over long sequences) the
// splits write their states to the workspace for a combine kernel.  Measured: 32 x 12 heads of 16,384 rows with weights 88 us for this kernel
// (453 MB of cache and 25 of scores, 84 % of the copy rate) and 22 for the combine kernel; 64 x 8 heads of 2,048
// rows 22-25 us; 8 x 8 float32 heads of 4,099 rows of 32 in one launch of clusters, 13 us with the host's part.
#include "attn_tc_common.cuh"
#include "kv4.cuh"
#include <math.h>

namespace attn {

constexpr int KD_WARPS = 4;
constexpr int KD_THREADS = KD_WARPS * 32;
constexpr int KD_WCHUNK = 4096;  // keys per combine CTA
constexpr int KD_SPLIT = 64 * KD_WARPS;  // keys a CTA takes at least, where there are so many
constexpr int KD_CLUSTER = 8;            // most CTAs of a cluster (the portable limit)
// A tile whose p s and p stay below these keeps its references.  A scale s counts as the power of two above it, 0 as
// the smallest of float16's, 2^-23, and one that is not finite as the largest: p reaches 2^39 only where p s as counted passes 2^15.  Sums of p stay far
// below float32's largest, and a reference lies at most 39 below and 16 above the largest score, so that what is
// flushed, 2^-126 of the reference, is nothing beside it.
constexpr float KD_MOST_P = 0x1p39f, KD_MOST_PS = 0x1p15f;
constexpr int KD_LEAST_SCALE = -23, KD_MOST_SCALE = 16;

struct Kv4Decode {
  const void* q;
  void* o;
  float* lse;
  const int* lengths;
  const float* w_in;
  float* w_out;
  int64_t q_sb, q_sh, o_sb, o_sh, w_sb, w_sh;
  int NH, NKV, G, L;
  int ns, per;     // splits, keys per split (a multiple of 64)
  int cluster;     // the splits are a cluster's CTAs
  int nq, chunks;  // query heads per CTA, and CTAs' chunks of them per key head
  float scale_log2;
  int alone;       // this kernel finishes o and lse
  float* states;  // [B*NH][ns][D + 2]: reference of p (log2 units), sum, unnormalised o; alone, [B*NH][2]: reference and sum
  float* scores;  // [B*NH][L]: scores in log2 units, where they do not fit beside the CTA's other shared memory
  int weights;    // whether weights are wanted
  int zsmem;      // the scores of the CTA's keys stay in shared memory
};

// The most splits a call's keys are cut into: rounds of a CTA's warps, at most KD_MOST_SPLITS.
constexpr int KD_MOST_SPLITS = 128;
static int kd_most_splits(int L) {
  const int rounds = (L + KD_SPLIT - 1) / KD_SPLIT;
  return rounds < KD_MOST_SPLITS ? rounds : KD_MOST_SPLITS;
}
// Scores that a CTA keeps in shared memory for the weights (16 KB).
constexpr int KD_ZFLOATS = 4096;

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The exponent of a normal number.
__device__ __forceinline__ int kd_exponent(float x) { return (int)(__float_as_uint(x) >> 23 & 255u) - 127; }

// max over the warp (NaN ignored)
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Where a code's bits stand in its float16: n * 2^-24 and, in the second nibble, 16 n * 2^-24; the second nibble
// for both, n * 2^-20; or the top of the mantissa, n * 2^-18.
enum KdPlace { KD_INPLACE, KD_SECOND, KD_TOP };
constexpr uint32_t KD_LOW = 0x000f000fu, KD_HIGH = 0x00f000f0u, KD_TOPMOST = 0x03c003c0u;
// Nibbles 2*PAIR and 2*PAIR + 1 of each half word as two float16 pairs (left shifts as products, which run
// beside the ANDs on the multiply-add pipe).
template <int PLACE, int PAIR>
__device__ __forceinline__ void kd_pairs(uint32_t w, uint32_t& a, uint32_t& b) {
  const uint32_t x = PAIR ? w >> 8 : w;
  if constexpr (PLACE == KD_TOP) {
    a = (x * 64u) & KD_TOPMOST;
    b = (x * 4u) & KD_TOPMOST;
  } else if constexpr (PLACE == KD_SECOND) {
    a = (x * 16u) & KD_HIGH;
    b = x & KD_HIGH;
  } else {
    a = x & KD_LOW;
    b = x & KD_HIGH;
  }
}
// c += (codes of two key rows) * (query): four codes a lane of each row.
template <int PLACE, int PAIR>
__device__ __forceinline__ void kd_score_mma(float (&c)[4], uint32_t wa, uint32_t wb, const uint32_t (&q)[2]) {
  uint32_t a0, a1, a2, a3;
  kd_pairs<PLACE, PAIR>(wa, a0, a2);
  kd_pairs<PLACE, PAIR>(wb, a1, a3);
  mma_f16(c, a0, a1, a2, a3, q[0], q[1]);
}
// acc += (codes of one value row pair) * (p s): x holds four elements of two keys, y of two more.
template <int PLACE, int PAIR>
__device__ __forceinline__ void kd_value_mma(float (&acc)[4], uint32_t x, uint32_t y, uint32_t b0, uint32_t b1) {
  uint32_t xa, xb, ya, yb;
  kd_pairs<PLACE, PAIR>(x, xa, xb);
  kd_pairs<PLACE, PAIR>(y, ya, yb);
  mma_f16(acc, xa, xb, ya, yb, b0, b1);
}

// Sizes of a warp's shared memory for head_dim D and NQ queries.
template <int D, int NQ, bool F32>
struct KdTile {
  static constexpr int TILE = D >= 128 ? 32 : 64;        // keys per warp step
  static constexpr int GROUPS = kv4_groups(D);
  static constexpr int COLS = F32 ? 2 * NQ : NQ;         // columns of the products
  static constexpr int CODE_BYTES = TILE * D / 2;        // one of K, V
  static constexpr int PARAM_BYTES = TILE * GROUPS * 4;
  static constexpr int STAGE = 2 * (CODE_BYTES + PARAM_BYTES);
  static constexpr int STAGES = D >= 64 ? 2 : 3;
  static constexpr int SC_LD = TILE + 4;                 // floats per query of the score tile (no bank conflicts)
  static constexpr int P_LD = TILE + 16;                 // halves per column of the p s tile (likewise)
  static constexpr int SC_BYTES = NQ * SC_LD * 4;
  static constexpr int P_BYTES = GROUPS * COLS * P_LD * 2;
  static constexpr int WARP = STAGES * STAGE + SC_BYTES + P_BYTES;
  static constexpr int Q_FLOATS = NQ * D + NQ * (1 + GROUPS);
  static constexpr int MERGE = (KD_WARPS + 1) * NQ * (D + 2) * 4;  // the warps' states and the CTA's, over the stages
  static constexpr int BYTES = KD_WARPS * WARP + Q_FLOATS * 4;
  static_assert(STAGE % 16 == 0 && SC_BYTES % 16 == 0 && P_BYTES % 16 == 0, "alignment");
  static_assert(MERGE <= KD_WARPS * WARP, "the merge reuses the stages");
};

__device__ __forceinline__ float kd_peer_load(uint32_t addr) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(addr) : "memory");
  return x;
}
// A float of CTA `rank` of the cluster, at the place of p in this CTA's shared memory.
__device__ __forceinline__ float kd_peer(const float* p, uint32_t rank) {
  return kd_peer_load(cluster_addr(p, rank));
}

// log(2^m l).  m and l's exponent, which nearly cancel, are added first: their sum is exact.
__device__ __forceinline__ float kd_lse(float m, float l) {
  if (!(l > 0.f || l != l)) return -INFINITY;
  const int e = kd_exponent(l);
  return (m + (float)e + log2f(ldexpf(l, -e))) * 0.6931471805599453f;
}

// Every thread of the cluster's CTAs: earlier writes are visible to the others after it.  All CTAs of a
// cluster are resident together and reach both of the kernel's syncs on every path.
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(KD_THREADS, D >= 128 ? 4 : NQ > 2 ? 4 : 5) kv4_decode_kernel(const Kv4View c, const Kv4Decode p) {
  constexpr bool F32 = sizeof(T) == 4;
  using S = KdTile<D, NQ, F32>;
  constexpr int GROUPS = S::GROUPS, GS = kv4_group(D), KD_TILE = S::TILE, PL = KD_TILE / 32;  // PL keys per lane
  constexpr int KPLACE = F32 ? KD_TOP : KD_SECOND, VPLACE = F32 ? KD_TOP : KD_INPLACE;
  // scores are formed again where the reference moves, in place of being kept in registers until then: eight queries
  // of head_dim 128 have none left (16 x 64 heads over 8 of up to 8,191 rows: 51.4 -> 48.5 us; elsewhere it costs up to 4 %)
  constexpr bool AGAIN = GROUPS == 2 && NQ == 8;
  // the largest p s after a move: low, p's arguments are small and rounded finely; high, small p s keep float16's bits
  constexpr float ROOM = F32 ? 3.f : 9.f;
  constexpr int MT = D / 16;   // 16-row tiles of the value product
  constexpr int KS = D / 16;   // 16-deep steps of the score product
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int g = lane / 4, t = lane % 4;
  uint8_t* ws = smem + warp * S::WARP;
  float* sc = reinterpret_cast<float*>(ws + S::STAGES * S::STAGE);
  __half* sp = reinterpret_cast<__half*>(ws + S::STAGES * S::STAGE + S::SC_BYTES);
  float* sq = reinterpret_cast<float*>(smem + KD_WARPS * S::WARP);  // [NQ][D]
  float* sfac = sq + NQ * D;                                        // [NQ]: score per unit of the product
  float* ssum = sfac + NQ;                                          // [NQ][GROUPS]: scale * sum of q
  grid_dependency_wait();
  grid_dependents_launch();
  const int split = blockIdx.x % p.ns;
  const int unit = blockIdx.x / p.ns;  // (sequence, key head, chunk of its query heads)
  const int chunk = unit % p.chunks, bk = unit / p.chunks;
  const int b = bk / p.NKV, kvh = bk % p.NKV;
  const int h0 = kvh * p.G + chunk * NQ, nq = min(NQ, p.G - chunk * NQ);
  const int n = seq_length(p.lengths, b, p.L);
  const int j0 = split * p.per, j1 = min(n, j0 + p.per);
  const int tiles = j1 > j0 ? (j1 - j0 + KD_TILE - 1) / KD_TILE : 0;
  const int64_t row0 = b * c.sb + kvh * c.sh;

  // tile i of this warp: keys j0 + (i * KD_WARPS + warp) * KD_TILE on, rows rounded up to 16 (the
  // capacity and the strides are multiples of 16 rows, so every copy is whole 16-byte pieces in bounds)
  auto fetch = [&](int i) {
    const int tile = i * KD_WARPS + warp;
    if (tile < tiles) {
      const int j = j0 + tile * KD_TILE;
      const int rows = min(KD_TILE, (j1 - j + 15) / 16 * 16);
      uint8_t* st = ws + (i % S::STAGES) * S::STAGE;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const int64_t row = which * c.si + row0 + j;
        const uint8_t* src = c.codes + row * (D / 2);
        uint8_t* dst = st + which * S::CODE_BYTES;
#pragma unroll
        for (int k = 0; k < (S::CODE_BYTES + 511) / 512; ++k)
          if ((k * 32 + lane) * 16 < rows * (D / 2)) cp_async16(dst + (k * 32 + lane) * 16, src + (k * 32 + lane) * 16);
        const uint8_t* psrc = reinterpret_cast<const uint8_t*>(c.params + row * GROUPS);
        uint8_t* pdst = st + 2 * S::CODE_BYTES + which * S::PARAM_BYTES;
        if (lane * 16 < rows * GROUPS * 4) cp_async16(pdst + lane * 16, psrc + lane * 16);
      }
    }
    cp_async_commit();
  };
  if (tiles == 0 && !p.alone) {  // a split behind its sequence's end
    for (int i = threadIdx.x; i < nq * (D + 2); i += KD_THREADS)
      p.states[(((int64_t)b * p.NH + h0 + i / (D + 2)) * p.ns + split) * (D + 2) + i % (D + 2)] = i % (D + 2) ? 0.f : -INFINITY;
    return;
  }
#pragma unroll
  for (int i = 0; i < S::STAGES - 1; ++i) fetch(i);

  // the queries: float32 rows, each row's power of two, its groups' sums
  for (int q = warp; q < NQ; q += KD_WARPS) {
    float big = 0.f, sum[GROUPS];
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) sum[k] = 0.f;
    float x[(D + 31) / 32];
#pragma unroll
    for (int k = 0; k < (D + 31) / 32; ++k) {
      const int d = k * 32 + lane;
      x[k] = q < nq && d < D ? Elem<T>::load((const T*)p.q + b * p.q_sb + (int64_t)(h0 + q) * p.q_sh + d) : 0.f;
      big = fmaxf(big, fabsf(x[k]));
      sum[k * 32 / GS] += x[k];
    }
    big = warp_max(big);
    // 2^(11 - exponent of the largest), so that the scaled row is below 2^12; exponents are kept to
    // where both powers are normal numbers (a row that reaches 2^122, whose scores float32 hardly holds, gives NaN)
    int e = (int)((__float_as_uint(big) >> 23) & 255u) - 127;
    e = min(max(e, -110), 118);
    const float up = __uint_as_float((uint32_t)(127 + 11 - e) << 23);
#pragma unroll
    for (int k = 0; k < (D + 31) / 32; ++k)
      if (k * 32 + lane < D) sq[q * D + k * 32 + lane] = x[k] * up;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
      const float total = warp_sum(sum[k]);
      if (lane == 0) ssum[q * GROUPS + k] = total * p.scale_log2;
    }
    // the product carries the codes' 2^-18 or 2^-20 and the row's `up`
    if (lane == 0) sfac[q] = p.scale_log2 * __uint_as_float((uint32_t)(127 + (F32 ? 7 : 9) + e) << 23);
  }
  __syncthreads();

  // B operand of the score product: column g holds query g (or part g % 2 of query g / 2), in the
  // order in which lane t finds the codes of its part of a row
  uint32_t qb[KS][2];
  {
    const int q = F32 ? g / 2 : g;
    const bool use = g < S::COLS;
    auto part = [&](float x) -> float {
      const float hi = __half2float(__float2half_rn(x));
      return F32 ? ((g & 1) ? x - hi : hi) : x;
    };
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      // lane t's codes: D / 4 elements per row in runs of min(D / 4, 16) (a run per group); step s
      // takes four of them: registers (e0, e1) and (e2, e3) at register-pair offsets
      int e0, e1, e2, e3;
      if constexpr (D >= 32) {
        const int per_group = GS / 4;                       // elements of a group per lane
        const int base = (s * 4 / per_group) * GS + t * per_group + (s * 4 % per_group) / 8 * 8;
        const int o = (s & 1) * 2;                          // word nibbles 0,4 | 1,5 then 2,6 | 3,7
        e0 = base + o; e1 = base + o + 4; e2 = base + o + 1; e3 = base + o + 5;
      } else {
        e0 = 4 * t; e1 = 4 * t + 2; e2 = 4 * t + 1; e3 = 4 * t + 3;
      }
      const float* row = sq + (use ? q : 0) * D;
      qb[s][0] = use ? pack_h2(part(row[e0]), part(row[e1])) : 0u;
      qb[s][1] = use ? pack_h2(part(row[e2]), part(row[e3])) : 0u;
    }
  }

  // scores kept for the weights: this CTA's keys in shared memory, or every key's in the workspace
  float* zrow = p.zsmem ? reinterpret_cast<float*>(smem + S::BYTES) - j0 : p.scores + ((int64_t)b * p.NH + h0) * p.L;
  const int64_t zld = p.zsmem ? p.per : p.L;

  float m[NQ], l[NQ], mg[NQ][GROUPS];
  float acc[MT][4];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    m[q] = -INFINITY;
    l[q] = 0.f;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) mg[q][k] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[i][k] = 0.f;
  // m: the reference that p is relative to (log2 units); head_dim 128's second group has one of its own, log2(ratio)
  // below it, so that its p are the first's times `ratio`
  float ratio[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) ratio[q] = 1.f;

  for (int i = 0; i * KD_WARPS + warp < tiles; ++i) {
    fetch(i + S::STAGES - 1);
    cp_async_wait<S::STAGES - 1>();
    __syncwarp();
    const uint8_t* st = ws + (i % S::STAGES) * S::STAGE;
    const __half2* kp = reinterpret_cast<const __half2*>(st + 2 * S::CODE_BYTES);
    const __half2* vp = kp + KD_TILE * GROUPS;
    const int j = j0 + (i * KD_WARPS + warp) * KD_TILE;

    // ---- scores: C[key][column] = sum over the row's codes ----
#pragma unroll
    for (int mt = 0; mt < KD_TILE / 16; ++mt) {
      float cs[GROUPS][4];
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) cs[k][0] = cs[k][1] = cs[k][2] = cs[k][3] = 0.f;
      const uint8_t* ra = st + (mt * 16 + g) * (D / 2);
      const uint8_t* rb = ra + 8 * (D / 2);
      if constexpr (D >= 32) {
        constexpr int WORDS = GS / 32;  // words of a group per lane
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
          uint32_t wa[WORDS], wb[WORDS];
          if constexpr (WORDS == 2) {
            const uint2 ua = *reinterpret_cast<const uint2*>(ra + k * 32 + t * 8);
            const uint2 ub = *reinterpret_cast<const uint2*>(rb + k * 32 + t * 8);
            wa[0] = ua.x; wa[1] = ua.y; wb[0] = ub.x; wb[1] = ub.y;
          } else {
            wa[0] = *reinterpret_cast<const uint32_t*>(ra + t * 4);
            wb[0] = *reinterpret_cast<const uint32_t*>(rb + t * 4);
          }
#pragma unroll
          for (int w = 0; w < WORDS; ++w) {
            const int s = (k * WORDS + w) * 2;
            kd_score_mma<KPLACE, 0>(cs[k], wa[w], wb[w], qb[s]);
            kd_score_mma<KPLACE, 1>(cs[k], wa[w], wb[w], qb[s + 1]);
          }
        }
      } else {
        // 4 codes per lane: byte 0 to the low half, byte 1 to the high half
        const uint32_t xa = __byte_perm(*reinterpret_cast<const uint16_t*>(ra + t * 2), 0, 0x4140);
        const uint32_t xb = __byte_perm(*reinterpret_cast<const uint16_t*>(rb + t * 2), 0, 0x4140);
        kd_score_mma<KPLACE, 0>(cs[0], xa, xb, qb[0]);
      }
      float r[4] = {cs[0][0], cs[0][1], cs[0][2], cs[0][3]};
      if constexpr (GROUPS == 2) {  // the groups' scales belong to the key: rows g and g + 8
        const float2 sa0 = __half22float2(kp[(mt * 16 + g) * 2]), sa1 = __half22float2(kp[(mt * 16 + g) * 2 + 1]);
        const float2 sb0 = __half22float2(kp[(mt * 16 + g + 8) * 2]), sb1 = __half22float2(kp[(mt * 16 + g + 8) * 2 + 1]);
        r[0] = sa0.x * cs[0][0] + sa1.x * cs[1][0];
        r[1] = sa0.x * cs[0][1] + sa1.x * cs[1][1];
        r[2] = sb0.x * cs[0][2] + sb1.x * cs[1][2];
        r[3] = sb0.x * cs[0][3] + sb1.x * cs[1][3];
      }
      if constexpr (F32) {  // a query's two parts are one lane's two columns
        if (t < NQ) {
          sc[t * S::SC_LD + mt * 16 + g] = r[0] + r[1];
          sc[t * S::SC_LD + mt * 16 + g + 8] = r[2] + r[3];
        }
      } else {
        if (2 * t < NQ) {
          sc[2 * t * S::SC_LD + mt * 16 + g] = r[0];
          sc[2 * t * S::SC_LD + mt * 16 + g + 8] = r[2];
        }
        if (2 * t + 1 < NQ) {
          sc[(2 * t + 1) * S::SC_LD + mt * 16 + g] = r[1];
          sc[(2 * t + 1) * S::SC_LD + mt * 16 + g + 8] = r[3];
        }
      }
    }
    __syncwarp();

    // ---- softmax: key lane of every 32 of the tile ----
    float ks[PL][GROUPS], km[PL][GROUPS], vs[PL][GROUPS], vm[PL][GROUPS];
    bool valid[PL];
#pragma unroll
    for (int u = 0; u < PL; ++u) {
      const int key = u * 32 + lane;
      valid[u] = j + key < j1;
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) {
        const float2 a = __half22float2(kp[key * GROUPS + k]), v = __half22float2(vp[key * GROUPS + k]);
        ks[u][k] = a.x; km[u][k] = a.y;
        vs[u][k] = valid[u] ? v.x : 0.f;
        vm[u][k] = valid[u] ? v.y : 0.f;
      }
    }
    auto score = [&](int q, int u) {
      const float raw = sc[q * S::SC_LD + u * 32 + lane] * sfac[q];
      float s = GROUPS == 1 ? raw * ks[u][0] : raw;
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) s = fmaf(km[u][k], ssum[q * GROUPS + k], s);
      return valid[u] ? s : -INFINITY;
    };
    float z[NQ][PL];
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int u = 0; u < PL; ++u) {
        z[q][u] = score(q, u);
        if (AGAIN && p.weights && valid[u] && q < nq) zrow[q * zld + j + u * 32 + lane] = z[q][u];
      }
    // p, and a lane's two p s of a query: of its key's two groups, or of its two keys (PL * GROUPS is 2)
    float e[NQ][PL], x[NQ][2], most_e = 0.f;
    __half2 h[NQ], most = __floats2half2_rn(0.f, 0.f);
    auto weigh = [&](int q) {
#pragma unroll
      for (int u = 0; u < PL; ++u) e[q][u] = valid[u] ? ex2_approx(z[q][u] - m[q]) : 0.f;
      x[q][0] = e[q][0] * vs[0][0];
      x[q][1] = GROUPS == 1 ? e[q][PL - 1] * vs[PL - 1][0] : e[q][0] * ratio[q] * vs[0][GROUPS - 1];
      h[q] = __floats2half2_rn(x[q][0], x[q][1]);
    };
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      weigh(q);
      most_e = fmax3(most_e, e[q][0], e[q][PL - 1]);  // (NaN ignored, here and below)
      most = __hmax2(most, h[q]);
    }
    if (__any_sync(0xffffffffu, !(most_e < KD_MOST_P && __low2float(most) < KD_MOST_PS && __high2float(most) < KD_MOST_PS))) {
      // (warp-uniform) new references, with room for p s to grow, and what was summed with the old ones
      float f[NQ][GROUPS];
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        if constexpr (AGAIN)
#pragma unroll
          for (int u = 0; u < PL; ++u) z[q][u] = score(q, u);
        float ref[GROUPS];
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
          const float old = k ? m[q] - lg2(ratio[q]) : m[q];
          float t = -INFINITY;
#pragma unroll
          for (int u = 0; u < PL; ++u)
            t = fmaxf(t, z[q][u] + (float)min(max(kd_exponent(vs[u][k]) + 1, KD_LEAST_SCALE), KD_MOST_SCALE));
          t = warp_max(t);
          ref[k] = t > old + 15.f ? t - ROOM : old;
        }
        f[q][0] = m[q] == -INFINITY ? 0.f : ex2_approx(m[q] - ref[0]);
        if constexpr (GROUPS == 2) {
          const float now = ref[0] == -INFINITY ? 1.f : ex2_approx(ref[0] - ref[1]);
          f[q][1] = f[q][0] * __fdividef(now, ratio[q]);
          ratio[q] = now;
        }
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) mg[q][k] *= f[q][0];
        m[q] = ref[0];
        l[q] *= f[q][0];
        weigh(q);
      }
      float c0[GROUPS], c1[GROUPS];  // of this lane's columns
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) {
        c0[k] = c1[k] = 1.f;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          if constexpr (F32) {
            if (t == q) c0[k] = c1[k] = f[q][k];
          } else {
            if (2 * t == q) c0[k] = f[q][k];
            if (2 * t + 1 == q) c1[k] = f[q][k];
          }
        }
      }
#pragma unroll
      for (int k = 0; k < MT; ++k) {
        constexpr int PER = MT / GROUPS;
        acc[k][0] *= c0[k / PER]; acc[k][1] *= c1[k / PER]; acc[k][2] *= c0[k / PER]; acc[k][3] *= c1[k / PER];
      }
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int u = 0; u < PL; ++u) {
        l[q] += e[q][u];
        if (!AGAIN && p.weights && valid[u] && q < nq) zrow[q * zld + j + u * 32 + lane] = z[q][u];
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) mg[q][k] = fmaf(e[q][u], vm[u][k], mg[q][k]);
      }
#pragma unroll
    for (int i2 = 0; i2 < 2; ++i2) {
      const int key = (GROUPS == 1 ? i2 * 32 : 0) + lane;
      // position of the key among its 16 in the B operand: lane t's four slots are keys t, t+4, t+8, t+12
      const int at = (key & ~15) + (key & 3) * 4 + ((key >> 2) & 3);
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const __half hi = i2 ? __high2half(h[q]) : __low2half(h[q]);
        __half* col = sp + ((GROUPS == 2 ? i2 : 0) * S::COLS + (F32 ? 2 * q : q)) * S::P_LD;
        col[at] = hi;
        if constexpr (F32) col[S::P_LD + at] = __float2half_rn((x[q][i2] - __half2float(hi)) * 2048.f);
      }
    }
    __syncwarp();

    // ---- values: acc[d][column] += sum over the keys of codes * p s ----
    // (the tensor core's additions round towards zero; a float32 output's tiles are added with rounding to nearest,
    // so that the bias of long sums stays below the other errors)
    const uint8_t* vc = st + S::CODE_BYTES;
    float tile_sum[F32 ? MT : 1][4];
    if constexpr (F32)
#pragma unroll
      for (int k = 0; k < MT; ++k) tile_sum[k][0] = tile_sum[k][1] = tile_sum[k][2] = tile_sum[k][3] = 0.f;
    float(*sum_v)[4] = F32 ? tile_sum : acc;
#pragma unroll
    for (int kk = 0; kk < KD_TILE / 16; ++kk) {
      const uint8_t* r0 = vc + (kk * 16 + t) * (D / 2);  // keys t, t+4, t+8, t+12
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) {
        uint32_t b0 = 0, b1 = 0;
        if (g < S::COLS) {
          const uint2 u = *reinterpret_cast<const uint2*>(sp + (k * S::COLS + g) * S::P_LD + kk * 16 + t * 4);
          b0 = u.x;
          b1 = u.y;
        }
        if constexpr (D >= 64) {
          const uint32_t w0 = *reinterpret_cast<const uint32_t*>(r0 + k * 32 + g * 4);
          const uint32_t w1 = *reinterpret_cast<const uint32_t*>(r0 + 4 * (D / 2) + k * 32 + g * 4);
          const uint32_t w2 = *reinterpret_cast<const uint32_t*>(r0 + 8 * (D / 2) + k * 32 + g * 4);
          const uint32_t w3 = *reinterpret_cast<const uint32_t*>(r0 + 12 * (D / 2) + k * 32 + g * 4);
          uint32_t x = __byte_perm(w0, w1, 0x5410), y = __byte_perm(w2, w3, 0x5410);  // elements 0..3
          kd_value_mma<VPLACE, 0>(sum_v[k * 4 + 0], x, y, b0, b1);
          kd_value_mma<VPLACE, 1>(sum_v[k * 4 + 1], x, y, b0, b1);
          x = __byte_perm(w0, w1, 0x7632); y = __byte_perm(w2, w3, 0x7632);  // elements 4..7
          kd_value_mma<VPLACE, 0>(sum_v[k * 4 + 2], x, y, b0, b1);
          kd_value_mma<VPLACE, 1>(sum_v[k * 4 + 3], x, y, b0, b1);
        } else if constexpr (D == 32) {
          auto half_word = [&](int key) { return (uint32_t)*reinterpret_cast<const uint16_t*>(r0 + key * (D / 2) + g * 2); };
          const uint32_t x = half_word(0) | half_word(4) << 16, y = half_word(8) | half_word(12) << 16;
          kd_value_mma<VPLACE, 0>(sum_v[0], x, y, b0, b1);
          kd_value_mma<VPLACE, 1>(sum_v[1], x, y, b0, b1);
        } else {
          auto byte = [&](int key) { return (uint32_t)r0[key * (D / 2) + g]; };
          const uint32_t x = byte(0) | byte(4) << 16, y = byte(8) | byte(12) << 16;
          kd_value_mma<VPLACE, 0>(sum_v[0], x, y, b0, b1);
        }
      }
    }
    if constexpr (F32)
#pragma unroll
      for (int k = 0; k < MT; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[k][r] += tile_sum[k][r];
    __syncwarp();  // the stage and the p s tile may be written again
  }
  cp_async_wait<0>();

  // ---- the warps' states: [warp][query][D + 2] over the stages ----
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    l[q] = warp_sum(l[q]);
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) mg[q][k] = warp_sum(mg[q][k]);
  }
  __syncthreads();
  float* merge = reinterpret_cast<float*>(smem) + warp * NQ * (D + 2);
  // the codes' 2^-18 or 2^-24 (16 times that in the odd rows)
  constexpr float DOWN = F32 ? 0x1p18f : 0x1p24f, DOWN_ODD = F32 ? 0x1p18f : 0x1p20f;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    if (lane == 0) {
      merge[q * (D + 2)] = m[q];
      merge[q * (D + 2) + 1] = l[q];
    }
    const bool mine = F32 ? t == q : t == q / 2;
    if (mine) {
      const float second = GROUPS == 2 ? 1.f / ratio[q] : 1.f;
#pragma unroll
      for (int k = 0; k < MT; ++k) {
        constexpr int PER = GS / 8;  // elements of a group per lane row g
        const int gr = k * 2 / PER, d = gr * GS + g * PER + (k * 2) % PER;
        const float lo = F32 ? fmaf(acc[k][1], 1.f / 2048.f, acc[k][0]) : (q & 1) ? acc[k][1] : acc[k][0];
        const float hi = F32 ? fmaf(acc[k][3], 1.f / 2048.f, acc[k][2]) : (q & 1) ? acc[k][3] : acc[k][2];
        const float by = gr ? second : 1.f;
        merge[q * (D + 2) + 2 + d] = fmaf(lo, DOWN * by, mg[q][gr]);
        merge[q * (D + 2) + 3 + d] = fmaf(hi, DOWN_ODD * by, mg[q][gr]);
      }
    }
  }
  __syncthreads();
  // ---- the CTA's state: [query][D + 2] behind the warps' ----
  const float* all = reinterpret_cast<const float*>(smem);
  float* own = reinterpret_cast<float*>(smem) + KD_WARPS * NQ * (D + 2);
  for (int i = threadIdx.x; i < nq * D; i += KD_THREADS) {
    const int q = i / D, d = i % D;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < KD_WARPS; ++w) mx = fmaxf(mx, all[(w * NQ + q) * (D + 2)]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < KD_WARPS; ++w) {
      const float* a = all + (w * NQ + q) * (D + 2);
      const float f = ex2_approx(a[0] - ref);
      sum = fmaf(a[1], f, sum);
      o = fmaf(a[2 + d], f, o);
    }
    float* to = !p.alone ? p.states + (((int64_t)b * p.NH + h0 + q) * p.ns + split) * (D + 2) : own + q * (D + 2);
    to[2 + d] = o;
    if (d == 0) {
      to[0] = mx;
      to[1] = sum;
    }
  }
  if (!p.alone) return;  // merged by the combine kernel

  // ---- merge over the cluster (or this CTA alone) ----
  if (p.cluster) cluster_sync();
  else __syncthreads();
  float* smx = sfac;  // [NQ] merged references, [NQ] reciprocal sums (the queries' factors are no longer needed)
  float* sinv = sfac + NQ;
  if (threadIdx.x < nq) {
    const float* a = own + threadIdx.x * (D + 2);
    float mx = -INFINITY, sum = 0.f;
    for (int r = 0; r < p.ns; ++r) mx = fmaxf(mx, p.cluster ? kd_peer(a, r) : a[0]);
    const float ref = mx == -INFINITY ? 0.f : mx;
    for (int r = 0; r < p.ns; ++r)
      sum = fmaf(p.cluster ? kd_peer(a + 1, r) : a[1], ex2_approx((p.cluster ? kd_peer(a, r) : a[0]) - ref), sum);
    smx[threadIdx.x] = ref;
    sinv[threadIdx.x] = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const int64_t bh = (int64_t)b * p.NH + h0 + threadIdx.x;
    if (split == 0 && p.lse) p.lse[bh] = kd_lse(ref, sum);
    if (split == 0 && p.weights && p.chunks > 1) {
      p.states[bh * 2] = ref;
      p.states[bh * 2 + 1] = sum;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x + split * KD_THREADS; i < nq * D; i += p.ns * KD_THREADS) {
    const int q = i / D, d = i % D;
    const float* a = own + q * (D + 2);
    float o = 0.f;
    for (int r = 0; r < p.ns; ++r)
      o = fmaf(p.cluster ? kd_peer(a + 2 + d, r) : a[2 + d], ex2_approx((p.cluster ? kd_peer(a, r) : a[0]) - smx[q]), o);
    Elem<T>::store((T*)p.o + b * p.o_sb + (h0 + q) * p.o_sh + d, o * sinv[q]);
  }
  if (p.weights && p.chunks == 1) {  // all of a key head's queries are this CTA's: the weights of this CTA's keys
    const int64_t w0 = b * p.w_sb + kvh * p.w_sh;
    const int end = split + 1 == p.ns ? p.L : min(p.L, j0 + p.per);
    for (int key = j0 + threadIdx.x; key < end; key += KD_THREADS) {
      float w = p.w_in ? p.w_in[w0 + key] : 0.f;
      float sum = 0.f;
      if (key < n)
#pragma unroll
        for (int q = 0; q < NQ; ++q)
          if (q < nq) sum = fmaf(ex2_approx(zrow[q * zld + key] - smx[q]), sinv[q], sum);
      p.w_out[w0 + key] = w + sum;
    }
  }
  if (p.cluster) cluster_sync();  // the others may still read this CTA's state
}

// Merge the splits' states and add the weights: a CTA takes KD_WCHUNK keys of one (sequence, key head), and
// its share of the outputs.  A warp finds a head's reference and sum, the splits on its lanes, so that a call
// waits for memory three times, not once per head and split.  16 keys a thread keep enough bytes in flight at two
// CTAs an SM (110 us for the long case's two kernels and 33 for the shared heads'; 8 keys and four CTAs 110 and 35,
// 4 and six 127 and 37); without weights there is little to hold, and six CTAs share an SM (64 x 8 heads of 2,048
// rows 25 -> 22 us).
constexpr int KC_THREADS = 256;
constexpr int KC_HEADS = 32;  // query heads at a time
template <typename T, int D, bool WEIGHTS>
__global__ void __launch_bounds__(KC_THREADS, WEIGHTS ? 2 : 6) kv4_decode_combine_kernel(const Kv4Decode p) {
  __shared__ float smx[KC_HEADS], sinv[KC_HEADS];
  grid_dependency_wait();
  grid_dependents_launch();
  const int wchunks = WEIGHTS ? (p.L + KD_WCHUNK - 1) / KD_WCHUNK : 1;
  const int bk = blockIdx.x / wchunks, chunk = blockIdx.x % wchunks;
  const int b = bk / p.NKV, kvh = bk % p.NKV;
  const int n = seq_length(p.lengths, b, p.L);
  const int j0 = chunk * KD_WCHUNK + threadIdx.x;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  constexpr int PER = WEIGHTS ? KD_WCHUNK / KC_THREADS : 1;
  const int64_t bh0 = (int64_t)b * p.NH + kvh * p.G, w0 = b * p.w_sb + kvh * p.w_sh;
  // what does not depend on the states is asked for first: the sums so far, and the first head's scores
  float w[PER], have[PER], z[PER];
  const float* zrow = p.scores + bh0 * p.L + j0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = j0 + i * KC_THREADS;
    w[i] = 0.f;
    have[i] = WEIGHTS && p.w_in && j < p.L ? p.w_in[w0 + j] : 0.f;
    z[i] = WEIGHTS && j < n ? zrow[i * KC_THREADS] : -INFINITY;
  }
  for (int g0 = 0; g0 < p.G; g0 += KC_HEADS) {
    const int heads = min(KC_HEADS, p.G - g0);
    __syncthreads();
    for (int g = warp; g < heads; g += KC_THREADS / 32) {
      const int64_t bh = bh0 + g0 + g;
      float mx, sum;
      if (p.alone) {
        mx = p.states[bh * 2];
        sum = p.states[bh * 2 + 1];
      } else {
        const float* st = p.states + bh * p.ns * (D + 2);
        float m = -INFINITY, l = 0.f;  // of this lane's splits
        for (int i = lane; i < p.ns; i += 32) {
          const float a = st[(int64_t)i * (D + 2)], c = st[(int64_t)i * (D + 2) + 1];
          const float nm = fmaxf(m, a), ref = nm == -INFINITY ? 0.f : nm;
          l = fmaf(l, ex2_approx(m - ref), c * ex2_approx(a - ref));
          m = nm;
        }
        mx = warp_max(m);
        if (mx == -INFINITY) mx = 0.f;
        sum = warp_sum(l * ex2_approx(m - mx));
      }
      if (lane == 0) {
        smx[g] = mx;
        sinv[g] = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        if (!p.alone && chunk == 0 && p.lse) p.lse[bh] = kd_lse(mx, sum);
      }
    }
    __syncthreads();
    if (!p.alone) {
      for (int i = chunk * KC_THREADS + threadIdx.x; i < heads * D; i += wchunks * KC_THREADS) {
        const int g = i / D, d = i % D;
        const float* st = p.states + (bh0 + g0 + g) * p.ns * (D + 2);
        float o = 0.f;
#pragma unroll 8
        for (int k = 0; k < p.ns; ++k) o = fmaf(st[(int64_t)k * (D + 2) + 2 + d], ex2_approx(st[(int64_t)k * (D + 2)] - smx[g]), o);
        Elem<T>::store((T*)p.o + b * p.o_sb + (kvh * p.G + g0 + g) * p.o_sh + d, o * sinv[g]);
      }
    }
    if (WEIGHTS) {
      for (int g = 0; g < heads; ++g) {
        const float mx = smx[g], inv = sinv[g];
        zrow += p.L;
        const bool more = g0 + g + 1 < p.G;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const float x = z[i];
          z[i] = more && j0 + i * KC_THREADS < n ? zrow[i * KC_THREADS] : -INFINITY;  // of the next head
          w[i] = fmaf(ex2_approx(x - mx), inv, w[i]);
        }
      }
    }
  }
  if (WEIGHTS) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = j0 + i * KC_THREADS;
      // (behind the rows w is 0 times the reciprocal sums, NaN where one of them is)
      if (j < p.L) p.w_out[w0 + j] = j < n ? have[i] + w[i] : have[i];
    }
  }
}

// How a call is cut up.
struct KdPlan {
  int nq, chunks, ns, per, cluster, alone, zsmem;  // alone: the first kernel finishes o and lse
  size_t states, scores;  // floats of workspace
};

static KdPlan kd_plan(int B, int NH, int NKV, int L, int D, int dtype, int weights) {
  KdPlan k;
  const int G = NH / NKV;
  // a product has eight columns: eight queries, or four float32 ones in two parts each
  const int most_q = dtype == ATTN_F32 ? 4 : 8;
  k.nq = G == 1 ? 1 : G == 2 ? 2 : G <= 4 || most_q == 4 ? 4 : 8;
  k.chunks = (G + k.nq - 1) / k.nq;
  // about seven CTAs for every SM, none with less than a round of its warps: measured for 384, 512 and 128 units,
  // ns = 3, 2 and 8 took 117, 22 and 50 us, half as many 129, 25 and 59, twice as many 115, 24 and 59.  Up to four
  // CTAs for every SM they form clusters, a power of two of CTAs up to eight, and the call is one launch.  An SM holds
  // four or five CTAs, and three where scores fill the shared memory of head_dim 128 or of eight queries; clusters that
  // find no room wait for a whole cluster's.  Measured at 4,096 keys, clusters and two kernels: float32,
  // head_dim 128, four queries, 64 units 21 and 25 us, 72 units 27 and 30 (of 2,048 keys 20.5 and 17.4); bfloat16,
  // head_dim 64, eight queries, 64 units 25 and 23, 72 units 25 and 27; one query, 72 units 12 and 15, 80 units
  // (where the rule takes two kernels) 12 and 15, 128 units 20 and 15; 384 units of 16,384 keys 137 and 117
  const int64_t units = (int64_t)B * NKV * k.chunks;
  const int sms = current_device_sms();
  const int64_t want = ((int64_t)sms * 7 + units / 2) / units > 1 ? ((int64_t)sms * 7 + units / 2) / units : 1;
  const int most = L <= KD_SPLIT ? 1 : kd_most_splits(L);
  int ns = (int)(want < most ? want : most);
  int c = 2;
  while (c < ns && c < KD_CLUSTER) c *= 2;
  k.cluster = ns > 1 && c * units <= 4 * sms && ns <= 2 * KD_CLUSTER;
  if (k.cluster) ns = c;
  const int tiles = (L + 63) / 64;
  k.per = (tiles + ns - 1) / ns * 64;
  k.ns = k.cluster ? ns : (L + k.per - 1) / k.per;
  k.alone = k.cluster || k.ns == 1;
  // where a key head's queries take more than one CTA (chunks), the combine kernel adds their weights
  k.zsmem = weights && k.alone && k.chunks == 1 && (int64_t)k.nq * k.per <= KD_ZFLOATS;
  k.states = k.alone ? (weights && k.chunks > 1 ? (size_t)B * NH * 2 : 0) : (size_t)B * NH * k.ns * (D + 2);
  k.states = (k.states + 3) / 4 * 4;
  k.scores = weights && !k.zsmem ? (size_t)B * NH * L : 0;
  return k;
}

template <typename T, int D, int NQ>
static int kv4_decode_q(const Kv4View& c, const Kv4Decode& p, int B, cudaStream_t s) {
  using S = KdTile<D, NQ, sizeof(T) == 4>;
  static_assert(S::BYTES + KD_ZFLOATS * 4 <= 227 * 1024, "shared memory");
  static CtxOnce attr;
  if (!set_smem_limit_once(kv4_decode_kernel<T, D, NQ>, S::BYTES + KD_ZFLOATS * 4, attr)) return ATTN_ERR_CUDA;
  const int64_t units = (int64_t)B * p.NKV * p.chunks;
  if (units * p.ns >= (int64_t)1 << 31) {
    set_error("attn_kv4_decode: B*NH*L is too large for one launch; split the batch into several calls");
    return ATTN_ERR_UNSUPPORTED;
  }
  const dim3 grid((unsigned)(units * p.ns)), block(KD_THREADS);
  const size_t smem = S::BYTES + (p.zsmem ? (size_t)NQ * p.per * 4 : 0);
  cudaError_t e = p.cluster ? launch_pdl_cluster(kv4_decode_kernel<T, D, NQ>, p.ns, grid, block, smem, s, c, p)
                            : launch_pdl(kv4_decode_kernel<T, D, NQ>, grid, block, smem, s, c, p);
  count_launch();
  if (int rc = check_launch("kv4_decode_kernel", e)) return rc;
  if (p.alone && !(p.weights && p.chunks > 1)) return ATTN_OK;
  const int wc = p.weights ? (p.L + KD_WCHUNK - 1) / KD_WCHUNK : 1;
  const dim3 cgrid((unsigned)wc * B * p.NKV), cblock(KC_THREADS);
  e = p.weights ? launch_pdl(kv4_decode_combine_kernel<T, D, true>, cgrid, cblock, 0, s, p)
                : launch_pdl(kv4_decode_combine_kernel<T, D, false>, cgrid, cblock, 0, s, p);
  count_launch();
  return check_launch("kv4_decode_combine_kernel", e);
}

template <typename T, int D>
static int kv4_decode_d(const Kv4View& c, const Kv4Decode& p, int B, cudaStream_t s) {
  switch (p.nq) {
    case 1: return kv4_decode_q<T, D, 1>(c, p, B, s);
    case 2: return kv4_decode_q<T, D, 2>(c, p, B, s);
    case 4: return kv4_decode_q<T, D, 4>(c, p, B, s);
  }
  return kv4_decode_q<T, D, sizeof(T) == 4 ? 4 : 8>(c, p, B, s);
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

extern "C" size_t attn_kv4_decode_workspace_size(int B, int NH, int NKV, int L, int D, int dtype, int weights) {
  if (B <= 0 || NH <= 0 || NKV <= 0 || NH % NKV || L <= 0 || D <= 0) return 0;
  const KdPlan k = kd_plan(B, NH, NKV, L, D, dtype, weights);
  return (k.states + k.scores) * sizeof(float);
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
  const RowSet w(L, B, w_sb, NKV, w_sh);
  ATTN_REQUIRE(!weights_out || w.apart, "attn_kv4_decode: rows of the weights must not overlap");
  ATTN_REQUIRE(!weights_in || weights_in == weights_out || !w.meets(weights_in, w, weights_out, 4),
               "attn_kv4_decode: weights_in and weights_out must be the same array or not overlap");
  ATTN_REQUIRE(RowSet(D, B, o_sb, NH, o_sh).apart, "attn_kv4_decode: rows of the output must not overlap");
  const KdPlan k = kd_plan(B, NH, NKV, L, D, dtype, weights_out != nullptr);
  const size_t need = (k.states + k.scores) * sizeof(float);
  if (need && (!workspace || workspace_bytes < need)) {
    set_error("attn_kv4_decode: workspace of %zu bytes required", need);
    return ATTN_ERR_WORKSPACE;
  }
  ATTN_REQUIRE(aligned(workspace, 16), "attn_kv4_decode: workspace must be 16-byte aligned");
  Kv4Decode p = {};
  p.q = q; p.o = o; p.lse = lse; p.lengths = lengths; p.w_in = weights_in; p.w_out = weights_out;
  p.q_sb = q_sb; p.q_sh = q_sh; p.o_sb = o_sb; p.o_sh = o_sh; p.w_sb = w_sb; p.w_sh = w_sh;
  p.NH = NH; p.NKV = NKV; p.G = NH / NKV; p.L = L;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.nq = k.nq; p.chunks = k.chunks; p.ns = k.ns; p.per = k.per; p.cluster = k.cluster; p.alone = k.alone; p.zsmem = k.zsmem;
  p.weights = weights_out != nullptr;
  p.states = (float*)workspace;
  p.scores = k.scores ? p.states + k.states : nullptr;
  return dtype == ATTN_BF16 ? kv4_decode_t<__nv_bfloat16>(c, p, B, D, as_stream(stream))
                            : kv4_decode_t<float>(c, p, B, D, as_stream(stream));
}
