// Accumulated attention weights of a prompt: for every key j of a key head,
//   w[j] = sum over the head's query heads and the queries i >= max(j, first_query), i < length, of
//          p_ij = exp(scale q_i . k_j - lse_i),
// the column sums of the causal softmax whose row statistics attn_fwd left in lse.  The T x T matrix
// (attn_probs, the reference's cache_attn_weights) is never stored.
//
// bfloat16 (head_dim to 64) and tf32 (to 32) run on the tensor cores: a CTA takes 128 keys and streams
// the queries past them in tiles of 128, S^T = K Q^T by tcgen05.mma into TMEM with the keys on the lanes, so
// that a thread owns one key and its sum needs no other thread.  Per score there is one multiply-add, one ex2
// and one addition: at 16 ex2 per clock and SM a 128 x 128 tile takes 1,024 cycles there, four times its
// MMA, so the special-function unit is the bound: 9,216 tiles (32 x 8 heads of 1,024 tokens) are 34 us of
// it.  Measured 59 us, the unit 55-60 % busy: a warp spends as long on waiting for scores, masks and moving on
// to the next tile as in its exponentials, and other warps fill that time only in part.  Three CTAs of one
// score tile each share an SM (59 us; two CTAs of two score tiles, the next tile's scores asked for before
// the last ones are summed, 62-64; four CTAs, whose 80 registers spill, 62; eight warps of half the columns,
// 61-69).  A polynomial exponential on the multiply-add pipe for an eighth to a half of the columns was
// slower (66-81 against 64), as is every instruction added here.
//
// Other shapes and float32 run on CUDA cores: a CTA takes 64 keys and streams the queries past them in tiles of
// 64, a thread forms 4 x 4 scores (two 16-byte shared-memory reads for 16 products), and the 16 threads of a
// key add up their sums at the end.  Tiles are loaded four elements at a time where rows are aligned for it (float32,
// 15 heads of 1,024 tokens at head_dim 128: 108 us by single elements, 70 by fours; 32 of 64: 101 and 78; their
// products alone are 28 us at the multiply-add rate).
#include "attn_tc_common.cuh"
#include "kv4.cuh"
#include <math.h>

namespace attn {

constexpr int KW_TILE = 64;       // keys, and queries, of a CUDA-core tile
constexpr int KW_LD = KW_TILE + 4;
constexpr int KW_THREADS = 256;

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

struct KwWork {
  KeyWeights p;
  int nt, parts, BK, units;  // key tiles, parts of a key tile's queries, B*NKV
  FastDiv by_bk, by_nkv, by_parts;
  float* partial;            // [parts][B*NKV][T] when parts > 1
  int* err;
};

// One unit of work: key tile jt of (b, kvh), query tiles [lo, lo + span) of each of the G query heads in
// turn, of which this part takes the steps [begin, end).  Units are ordered longest first (the first
// key tiles) and dealt to the CTAs forth and back, which evens out their totals: 32 x 8 heads of 8 tiles
// come to 20 .. 22 tiles for each of 444 CTAs, dealt round and round to 17 .. 25.
struct KwUnit {
  int b, kvh, jt, part, n, lo, span, begin, end;
  __device__ __forceinline__ bool set(const KwWork& a, int round) {
    const int u = round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    if (u >= a.units) {
      begin = end = 0;
      return false;
    }
    open(a, u, AT_TILE);
    return true;
  }
  __device__ __forceinline__ void open(const KwWork& a, int u, int tile) {
    const uint32_t level = a.by_bk.div(u), bk = u - level * a.BK;
    jt = a.by_parts.div(level);
    part = level - jt * a.parts;
    b = a.by_nkv.div(bk);
    kvh = bk - b * a.p.NKV;
    n = seq_length(a.p.lengths, b, a.p.T);
    lo = max(jt, a.p.first / tile);
    span = max((n + tile - 1) / tile - lo, 0);
    const int total = span * a.p.G;
    begin = 0;
    end = total;
    if (a.parts > 1) {
      begin = (int)((int64_t)total * part / a.parts);
      end = (int)((int64_t)total * (part + 1) / a.parts);
    }
  }
};

// The query tiles of a unit in order: query head g of the key head, tile it.
struct KwSteps {
  int g, it;
  __device__ __forceinline__ void start(const KwUnit& w) {
    g = w.begin ? w.begin / max(w.span, 1) : 0;
    it = w.lo + w.begin - g * w.span;
  }
  __device__ __forceinline__ void next(const KwUnit& w) {
    if (++it == w.lo + w.span) {
      it = w.lo;
      ++g;
    }
  }
};

// The sum of key j of a unit: an output, or a part of one.
__device__ __forceinline__ void kw_write(const KwWork& a, const KwUnit& w, int j, float sum) {
  if (a.parts > 1) {
    a.partial[((int64_t)w.part * a.BK + (int64_t)w.b * a.p.NKV + w.kvh) * a.p.T + j] = sum;
  } else {
    const int64_t at = w.b * a.p.w_sb + w.kvh * a.p.w_sh + j;
    a.p.w_out[at] = (a.p.w_in ? a.p.w_in[at] : 0.f) + sum;
  }
}

// Rows [r0, r0 + 64) of a head, rows past `rows` as zeros, into sm[d][row].  Consecutive threads read consecutive
// elements; a thread steps from one to its next by (rows, elements) = (KW_THREADS / D, KW_THREADS % D).
template <typename T, bool TF32>
__device__ __forceinline__ void kw_load_tile(float* sm, const T* base, int64_t st, int r0, int rows, int D, int dr, int dd) {
  int r = threadIdx.x / D, d = threadIdx.x - r * D;
#pragma unroll 4
  for (; r < KW_TILE;) {
    const float x = r0 + r < rows ? Elem<T>::load(base + (int64_t)(r0 + r) * st + d) : 0.f;
    sm[d * KW_LD + r] = TF32 ? tf32_cut(x) : x;
    r += dr;
    d += dd;
    if (d >= D) {
      d -= D;
      ++r;
    }
  }
}

// The same where every fourth element of a row is aligned for four: a thread takes one row, every fourth quad of it, so
// that a warp reads 64 bytes (float32) of 8 rows at a time, and has all its loads in flight.
template <typename T, bool TF32>
__device__ __forceinline__ void kw_load_tile4(float* sm, const T* base, int64_t st, int r0, int rows, int D) {
  static_assert(KW_THREADS == 4 * KW_TILE, "a row per four threads");
  const int r = threadIdx.x / 4, d0 = threadIdx.x % 4 * 4;
  const bool in = r0 + r < rows;
  const T* src = base + (int64_t)(r0 + r) * st + d0;
  float4 x[8];  // head_dim up to 128
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k * 16 + d0 < D) x[k] = in ? load4(src + k * 16) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k * 16 + d0 < D) {
      float* to = sm + (k * 16 + d0) * KW_LD + r;
      to[0] = TF32 ? tf32_cut(x[k].x) : x[k].x;
      to[KW_LD] = TF32 ? tf32_cut(x[k].y) : x[k].y;
      to[2 * KW_LD] = TF32 ? tf32_cut(x[k].z) : x[k].z;
      to[3 * KW_LD] = TF32 ? tf32_cut(x[k].w) : x[k].w;
    }
}

template <typename T, bool TF32, bool VEC>
__global__ void __launch_bounds__(KW_THREADS) key_weights_simt_kernel(const KwWork a) {
  const KeyWeights& p = a.p;
  extern __shared__ __align__(16) float sm[];
  float* sk = sm;                    // [D][KW_LD]
  float* sq = sk + p.D * KW_LD;      // [D][KW_LD]
  float* sl = sq + p.D * KW_LD;      // [KW_TILE] -lse in log2 units
  grid_dependency_wait();
  grid_dependents_launch();
  KwUnit w;
  w.open(a, blockIdx.x, KW_TILE);
  const int dr = KW_THREADS / p.D, dd = KW_THREADS - dr * p.D;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;  // queries 4 tx.., keys 4 ty..
  const int j0 = w.jt * KW_TILE;
  auto load = [&](float* to, const void* from, int64_t at, int64_t stride, int r0) {
    if constexpr (VEC) kw_load_tile4<T, TF32>(to, (const T*)from + at, stride, r0, w.n, p.D);
    else kw_load_tile<T, TF32>(to, (const T*)from + at, stride, r0, w.n, p.D, dr, dd);
  };
  if (w.begin < w.end) load(sk, p.k, w.b * p.k_sb + w.kvh * p.k_sh, p.k_st, j0);
  float total[4] = {0.f, 0.f, 0.f, 0.f};
  KwSteps st;
  st.start(w);
  for (int i = w.begin; i < w.end; ++i, st.next(w)) {
    const int h = w.kvh * p.G + st.g, i0 = st.it * KW_TILE;
    __syncthreads();
    load(sq, p.q, w.b * p.q_sb + h * p.q_sh, p.q_st, i0);
    if (threadIdx.x < KW_TILE)
      sl[threadIdx.x] = i0 + threadIdx.x < w.n ? p.lse[((int64_t)w.b * p.NH + h) * p.T + i0 + threadIdx.x] * -1.4426950408889634f : 0.f;
    __syncthreads();
    float acc[4][4];
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) acc[x][y] = 0.f;
#pragma unroll 4
    for (int d = 0; d < p.D; ++d) {
      const float4 kv = *reinterpret_cast<const float4*>(sk + d * KW_LD + 4 * ty);
      const float4 qv = *reinterpret_cast<const float4*>(sq + d * KW_LD + 4 * tx);
      const float k4[4] = {kv.x, kv.y, kv.z, kv.w}, q4[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = fmaf(k4[x], q4[y], acc[x][y]);
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      float sum = 0.f;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int q = i0 + 4 * tx + y;
        const bool use = q < w.n && q >= p.first && q >= j0 + 4 * ty + x;
        const float e = ex2_approx(fmaf(acc[x][y], p.scale_log2, sl[4 * tx + y]));
        sum += use ? e : 0.f;
      }
      total[x] += sum;
    }
  }
#pragma unroll
  for (int off = 8; off > 0; off >>= 1)
#pragma unroll
    for (int x = 0; x < 4; ++x) total[x] += __shfl_xor_sync(0xffffffffu, total[x], off);
  if (tx < 4) {  // thread tx of a key group writes key tx
    const int j = j0 + 4 * ty + tx;
    if (j < p.T) {
      const float mine = tx == 0 ? total[0] : tx == 1 ? total[1] : tx == 2 ? total[2] : total[3];
      kw_write(a, w, j, j < w.n ? mine : 0.f);
    }
  }
}

// ---- tensor cores ------------------------------------------------------------------------------
constexpr int KT_CTAS = 3;                   // CTAs per SM
constexpr int KT_STAGES = 2;                 // query tiles in flight
constexpr int KT_KEYS = 2;                   // key tiles in flight
constexpr int KT_BUFS = 1;                   // score tiles in TMEM
constexpr int KT_THREADS = 192;              // 4 warps of sums, a TMA warp, an MMA warp
constexpr int KT_TMEM = KT_BUFS * AT_TILE;
constexpr int KT_SMEM = 1024 + (KT_KEYS + KT_STAGES) * AT_TILE_BYTES + 4 * AT_TILE * 4 + 256;

struct KwMaps {
  TileMap q, k;
};

struct KwBars {
  uint64_t k_full[KT_KEYS], k_empty[KT_KEYS], q_full[KT_STAGES], q_empty[KT_STAGES], s_full[KT_BUFS], s_free[KT_BUFS];
  uint32_t tmem;
};

// All query tiles of a CTA's units in order.
struct KwTiles {
  KwUnit w;
  KwSteps st;
  int i, round;
  bool more;
  __device__ __forceinline__ void open(const KwWork& a) {  // the first tile of the next unit that has one
    do more = w.set(a, round++);
    while (more && w.begin >= w.end);
    i = w.begin;
    if (more) st.start(w);
  }
  __device__ __forceinline__ void start(const KwWork& a) {
    round = 0;
    open(a);
  }
  __device__ __forceinline__ void next(const KwWork& a) {
    st.next(w);
    if (++i == w.end) open(a);
  }
};

// Two float32 in one register pair: sm_100's packed multiply-add and addition halve the issue slots.
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ void add2(uint64_t& a, uint64_t b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a) : "l"(b));
}
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x) {
  return pair(__float_as_uint(ex2_approx(__uint_as_float((uint32_t)x))),
              __float_as_uint(ex2_approx(__uint_as_float((uint32_t)(x >> 32)))));
}
__device__ __forceinline__ float pair_sum(uint64_t x) {
  return __uint_as_float((uint32_t)x) + __uint_as_float((uint32_t)(x >> 32));
}

// Wait for a load that is known to be in flight, after a wait elsewhere gave up: at most 0.1 s.
__device__ __forceinline__ void drain_load(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait_sleep(bar, parity, 200000u))
    if (globaltimer_ns() - t0 > 100000000ull) return;
}

template <bool TF32>
__global__ void __launch_bounds__(KT_THREADS, KT_CTAS)
key_weights_tc_kernel(const __grid_constant__ KwMaps maps, const KwWork a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;                                   // [KT_KEYS]
  uint8_t* sQ = sK + KT_KEYS * AT_TILE_BYTES;           // [KT_STAGES]
  float* sL = reinterpret_cast<float*>(sQ + KT_STAGES * AT_TILE_BYTES);  // [4 warps][128]
  KwBars* bars = reinterpret_cast<KwBars*>(sL + 4 * AT_TILE);
  const WaitErr werr = wait_err(a.err);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < KT_KEYS; ++i) {
      mbar_init(&bars->k_full[i], 1);
      mbar_init(&bars->k_empty[i], 1);
    }
    for (int i = 0; i < KT_BUFS; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->s_free[i], 4);
    }
    for (int i = 0; i < KT_STAGES; ++i) {
      mbar_init(&bars->q_full[i], 1);
      mbar_init(&bars->q_empty[i], 1);
    }
    fence_mbar_init();
  }
  if (warp == 5) {
    tmem_alloc(&bars->tmem, KT_TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  grid_dependency_wait();
  grid_dependents_launch();

  if (warp == 4) {
    // ---------------- TMA ----------------
    if (lane == 0) {
      int ku = 0, qn = 0;
      bool ok = true;
      KwUnit w;
      for (int round = 0; ok && w.set(a, round); ++round) {
        if (w.begin >= w.end) continue;
        const int ks = ku % KT_KEYS;
        if (!mbar_wait(&bars->k_empty[ks], ((ku / KT_KEYS) & 1) ^ 1, werr, 501)) { ok = false; break; }
        mbar_arrive_expect_tx(&bars->k_full[ks], AT_TILE_BYTES);
        load_tile(sK + ks * AT_TILE_BYTES, maps.k, &bars->k_full[ks], w.b, w.kvh, w.jt * AT_TILE);
        ++ku;
        KwSteps st;
        st.start(w);
        for (int i = w.begin; i < w.end; ++i, ++qn, st.next(w)) {
          const int qs = qn % KT_STAGES;
          if (!mbar_wait(&bars->q_empty[qs], ((qn / KT_STAGES) & 1) ^ 1, werr, 502)) { ok = false; break; }
          mbar_arrive_expect_tx(&bars->q_full[qs], AT_TILE_BYTES);
          load_tile(sQ + qs * AT_TILE_BYTES, maps.q, &bars->q_full[qs], w.b, w.kvh * a.p.G + st.g,
                    st.it * AT_TILE);
        }
      }
      if (!ok) {  // leave no load of this CTA's behind
        for (int i = max(0, ku - KT_KEYS); i < ku; ++i) drain_load(&bars->k_full[i % KT_KEYS], (i / KT_KEYS) & 1);
        for (int i = max(0, qn - KT_STAGES); i < qn; ++i) drain_load(&bars->q_full[i % KT_STAGES], (i / KT_STAGES) & 1);
      }
    }
  } else if (warp == 5) {
    // ---------------- MMA ----------------
    if (lane == 0) {
      const uint32_t idesc = TF32 ? idesc_tf32_f32(128, 128, 0, 0) : idesc_bf16_f32(128, 128, 0, 0);
      int ku = 0, qn = 0;
      bool ok = true;
      KwUnit w;
      for (int round = 0; ok && w.set(a, round); ++round) {
        if (w.begin >= w.end) continue;
        const int ks = ku % KT_KEYS;
        if (!mbar_wait(&bars->k_full[ks], (ku / KT_KEYS) & 1, werr, 503)) break;
        const uint64_t k_desc = smem_desc_sw128(smem_u32(sK + ks * AT_TILE_BYTES), 16, 1024);
        const int last = qn + w.end - w.begin;
        for (int t = qn; t < last; ++t) {
          const int qs = t % KT_STAGES, buf = t % KT_BUFS;
          if (!mbar_wait(&bars->q_full[qs], (t / KT_STAGES) & 1, werr, 504) ||
              !mbar_wait(&bars->s_free[buf], ((t / KT_BUFS) & 1) ^ 1, werr, 505)) { ok = false; break; }
          tc_fence_after();
          const uint64_t q_desc = smem_desc_sw128(smem_u32(sQ + qs * AT_TILE_BYTES), 16, 1024);
#pragma unroll
          for (int k = 0; k < AT_D / 16; ++k) {
            if constexpr (TF32)
              umma_ss_tf32(tmem + buf * 128, desc_step(k_desc, k * 32), desc_step(q_desc, k * 32), idesc, k > 0 ? 1u : 0u);
            else
              umma_ss(tmem + buf * 128, desc_step(k_desc, k * 32), desc_step(q_desc, k * 32), idesc, k > 0 ? 1u : 0u);
          }
          umma_commit(&bars->s_full[buf]);
          umma_commit(&bars->q_empty[qs]);
        }
        if (ok) umma_commit(&bars->k_empty[ks]);
        qn = last;
        ++ku;
      }
    }
  } else {
    // ---------------- sums: thread = key ----------------
    float* lb = sL + warp * AT_TILE;
    const uint32_t tS = tmem + ((uint32_t)(warp * 32) << 16);
    const uint64_t cpair = pair(__float_as_uint(a.p.scale_log2), __float_as_uint(a.p.scale_log2));
    const int row = warp * 32 + lane;
    bool ok = true;
    KwTiles ahead;          // the tile whose lse is in `next`
    float next[4];
    ahead.start(a);
    auto fetch = [&]() {
      if (!ahead.more) return;
      const int i0 = ahead.st.it * AT_TILE + lane;
      const float* src = a.p.lse + ((int64_t)ahead.w.b * a.p.NH + ahead.w.kvh * a.p.G + ahead.st.g) * a.p.T + i0;
#pragma unroll
      for (int k = 0; k < 4; ++k) next[k] = i0 + k * 32 < ahead.w.n ? src[k * 32] : 0.f;
    };
    fetch();
    int qn = 0;             // tiles summed
    KwUnit w;
    for (int round = 0; ok && w.set(a, round); ++round) {
      const int j = w.jt * AT_TILE + row;
      const int64_t at = w.b * a.p.w_sb + w.kvh * a.p.w_sh + j;
      const float have = a.parts == 1 && a.p.w_in && j < a.p.T ? a.p.w_in[at] : 0.f;
      float total = 0.f;
      KwSteps st;
      st.start(w);
      for (int i = w.begin; i < w.end; ++i, ++qn, st.next(w)) {
        const int buf = qn % KT_BUFS, i0 = st.it * AT_TILE;
        // -lse in log2 units for this warp; the next tile's is on its way while this one is summed
#pragma unroll
        for (int k = 0; k < 4; ++k) lb[k * 32 + lane] = next[k] * -LOG2E;
        ahead.next(a);
        fetch();
        __syncwarp();
        if (!__all_sync(0xffffffffu, mbar_wait(&bars->s_full[buf], (qn / KT_BUFS) & 1, werr, 506))) { ok = false; break; }
        tc_fence_after();
        // columns that count for this key: queries from max(j, first) to n - 1; the warp's bounds
        const int c0 = max(j, a.p.first) - i0, c1 = w.n - i0;
        const int c0_any = max(j - lane, a.p.first) - i0, c0_all = max(j - lane + 31, a.p.first) - i0;
        uint64_t sum[2] = {0, 0};  // four running sums of the tile as two packed pairs
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t x[32];
          tmem_ld32(tS + buf * 128 + cc * 32, x);
          tmem_wait_ld();
          if (cc == 3) {  // the scores are in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->s_free[buf]);
          }
          if (cc * 32 + 32 <= c0_any) continue;  // before every lane's first query
          const ulonglong2* l2 = reinterpret_cast<const ulonglong2*>(lb + cc * 32);
          uint64_t y[16];  // the exponentials' arguments
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const ulonglong2 l = l2[k];
            y[2 * k] = fma2(pair(x[4 * k], x[4 * k + 1]), cpair, l.x);
            y[2 * k + 1] = fma2(pair(x[4 * k + 2], x[4 * k + 3]), cpair, l.y);
          }
          if (cc * 32 < c0_all || cc * 32 + 32 > c1) {
            // the whole argument is replaced (by -inf, whose exponential is 0): where a column does not count, the
            // score, the query's lse and the scale's sign may be anything
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const int c = cc * 32 + 2 * k;
              y[k] = pair(c < c0 || c >= c1 ? 0xff800000u : (uint32_t)y[k],
                          c + 1 < c0 || c + 1 >= c1 ? 0xff800000u : (uint32_t)(y[k] >> 32));
            }
          }
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            add2(sum[0], ex2_pair(y[k]));
            add2(sum[1], ex2_pair(y[k + 1]));
          }
        }
        total += pair_sum(sum[0]) + pair_sum(sum[1]);
        __syncwarp();  // lb is written again for the next tile
      }
      if (!ok) break;
      if (j < a.p.T) {
        const float sum = j < w.n ? total : 0.f;
        if (a.parts > 1) a.partial[((int64_t)w.part * a.BK + (int64_t)w.b * a.p.NKV + w.kvh) * a.p.T + j] = sum;
        else a.p.w_out[at] = have + sum;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, KT_TMEM);
  }
}

__global__ void __launch_bounds__(256) key_weights_join_kernel(const KwWork a) {
  grid_dependency_wait();
  grid_dependents_launch();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)a.BK * a.p.T) return;
  const int bk = (int)(i / a.p.T), j = (int)(i - (int64_t)bk * a.p.T);
  float sum = 0.f;
  for (int k = 0; k < a.parts; ++k) sum += a.partial[((int64_t)k * a.BK + bk) * a.p.T + j];
  const int64_t at = bk / a.p.NKV * a.p.w_sb + bk % a.p.NKV * a.p.w_sh + j;
  a.p.w_out[at] = (a.p.w_in ? a.p.w_in[at] : 0.f) + sum;
}

// Parts that a key tile's queries are cut into: one from 592 units on, four for every SM of 148; below that enough
// for 1,184, and none of fewer than four query tiles (the parts cost a second launch, as long as a tile or two).
// The tensor-core kernel keeps 444 CTAs, the other one about as many.  Measured, one part and two, tiles of
// 128 (bfloat16, head_dim 64): 1,024 tokens, 384 units 21.5 and 19.4 us, 512 units 22.5 and 22.2, 576 units 22.5
// and 24.2, 640 units 22.2 and 27.7; 2,048 tokens, 512 units 40.1 and 34.6 (three 38.2), 640 units 38.2 and 39.9.  Of
// 64 (float32): 1,024 tokens, 512 units 105 and 77, 768 units 108 and 109, 1,024 units 139 and 143.
constexpr int KW_ENOUGH = 592;
static int key_weights_parts(int B, int NKV, int T, int tile) {
  const int64_t tiles = (T + tile - 1) / tile, units = (int64_t)B * NKV * tiles;
  if (units >= KW_ENOUGH) return 1;
  const int64_t parts = (2 * KW_ENOUGH + units - 1) / units;
  const int64_t most = tiles / 4 > 1 ? tiles / 4 : 1;
  return (int)(parts < most ? parts : most);
}

// What both kernels take beside the arguments.
static KwWork kw_work(const KeyWeights& p, int B, int tile, float* partial) {
  KwWork a;
  a.p = p;
  a.nt = (p.T + tile - 1) / tile;
  a.parts = key_weights_parts(B, p.NKV, p.T, tile);
  a.BK = B * p.NKV;
  a.units = a.BK * a.nt * a.parts;
  a.by_bk.set(a.BK);
  a.by_nkv.set(p.NKV);
  a.by_parts.set(a.parts);
  a.partial = partial;
  a.err = nullptr;
  return a;
}

static int key_weights_join(const KwWork& a, cudaStream_t s) {
  if (a.parts == 1) return ATTN_OK;
  const int64_t n = (int64_t)a.BK * a.p.T;
  const cudaError_t e = launch_pdl(key_weights_join_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
  count_launch();
  return check_launch("key_weights_join_kernel", e);
}

static int key_weights_simt(const KeyWeights& p, int B, int dtype, float* partial, cudaStream_t s) {
  const size_t smem = ((size_t)2 * p.D * KW_LD + KW_TILE) * sizeof(float);
  // four elements at a time where every row's quads are aligned for it
  const int64_t st[6] = {p.q_sb, p.q_st, p.q_sh, p.k_sb, p.k_st, p.k_sh};
  const size_t quad = dtype == ATTN_BF16 ? 8 : 16;
  bool vec = p.D % 4 == 0 && aligned(p.q, quad) && aligned(p.k, quad);
  for (int i = 0; i < 6; ++i) vec = vec && st[i] % 4 == 0;
  static CtxOnce attr[6];
  const int which = (dtype == ATTN_BF16 ? 0 : dtype == ATTN_TF32 ? 2 : 4) + vec;
  void (*const kernels[6])(KwWork) = {
      key_weights_simt_kernel<__nv_bfloat16, false, false>, key_weights_simt_kernel<__nv_bfloat16, false, true>,
      key_weights_simt_kernel<float, true, false>, key_weights_simt_kernel<float, true, true>,
      key_weights_simt_kernel<float, false, false>, key_weights_simt_kernel<float, false, true>};
  auto kern = kernels[which];
  if (!set_smem_limit_once(kern, (2 * 128 * KW_LD + KW_TILE) * 4, attr[which])) return ATTN_ERR_CUDA;
  const KwWork a = kw_work(p, B, KW_TILE, partial);
  const cudaError_t e = launch_pdl(kern, dim3((unsigned)a.units), dim3(KW_THREADS), smem, s, a);
  count_launch();
  if (int rc = check_launch("key_weights_simt_kernel", e)) return rc;
  return key_weights_join(a, s);
}

static bool key_weights_tc_ok(const KeyWeights& p, int dtype) {
  const int64_t q[3] = {p.q_sb, p.q_st, p.q_sh}, k[3] = {p.k_sb, p.k_st, p.k_sh};
  if (!aligned(p.q, 16) || !aligned(p.k, 16)) return false;
  for (int i = 0; i < 3; ++i)
    if (q[i] <= 0 || k[i] <= 0) return false;  // broadcast axes have no tensor map
  if (dtype == ATTN_TF32)
    return tc_head_dim_ok_tf32(p.D) && head_strides_ok_f32(q[0], q[1], q[2], p.D) && head_strides_ok_f32(k[0], k[1], k[2], p.D);
  return dtype == ATTN_BF16 && tc_head_dim_ok(p.D) && head_strides_ok(q[0], q[1], q[2], p.D) &&
         head_strides_ok(k[0], k[1], k[2], p.D);
}

static int key_weights_tc(const KeyWeights& p, int B, int tf32, float* partial, cudaStream_t s) {
  KwMaps maps;
  if (tf32) {
    if (!make_head_map_f32(&maps.q, p.q, B, p.NH, p.T, p.D, p.q_sb, p.q_st, p.q_sh, 128) ||
        !make_head_map_f32(&maps.k, p.k, B, p.NKV, p.T, p.D, p.k_sb, p.k_st, p.k_sh, 128))
      return ATTN_ERR_CUDA;
  } else if (!make_head_map(&maps.q, p.q, B, p.NH, p.T, p.D, p.q_sb, p.q_st, p.q_sh) ||
             !make_head_map(&maps.k, p.k, B, p.NKV, p.T, p.D, p.k_sb, p.k_st, p.k_sh)) {
    return ATTN_ERR_CUDA;
  }
  KwWork a = kw_work(p, B, AT_TILE, partial);
  a.err = dev_error_ptr();
  if (!a.err) return ATTN_ERR_CUDA;
  const int64_t ctas = KT_CTAS * (int64_t)current_device_sms();
  const unsigned grid = (unsigned)(a.units < ctas ? a.units : ctas);
  static CtxOnce attr[2];
  if (!(tf32 ? set_smem_limit_once(key_weights_tc_kernel<true>, KT_SMEM, attr[1])
             : set_smem_limit_once(key_weights_tc_kernel<false>, KT_SMEM, attr[0])))
    return ATTN_ERR_CUDA;
  cudaError_t e = tf32 ? launch_pdl(key_weights_tc_kernel<true>, dim3(grid), dim3(KT_THREADS), KT_SMEM, s, maps, a)
                       : launch_pdl(key_weights_tc_kernel<false>, dim3(grid), dim3(KT_THREADS), KT_SMEM, s, maps, a);
  count_launch();
  if (int rc = check_launch("key_weights_tc_kernel", e)) return rc;
  return key_weights_join(a, s);
}

}  // namespace attn

using namespace attn;

extern "C" size_t attn_key_weights_workspace_size(int B, int NKV, int T) {
  if (B <= 0 || NKV <= 0 || T <= 0 || T > 1 << 30) return 0;
  // whichever kernel the tensors suit
  const int tc = key_weights_parts(B, NKV, T, AT_TILE), simt = key_weights_parts(B, NKV, T, KW_TILE);
  const int parts = tc > simt ? tc : simt;
  return parts > 1 ? (size_t)parts * B * NKV * T * sizeof(float) : 0;
}

extern "C" int attn_key_weights(const void* q, const void* k, const float* lse, const float* weights_in,
                                float* weights_out, int B, int NH, int NKV, int T, int D, int64_t q_sb, int64_t q_st,
                                int64_t q_sh, int64_t k_sb, int64_t k_st, int64_t k_sh, int64_t w_sb, int64_t w_sh,
                                int first_query, const int* lengths, float scale, int dtype, void* workspace,
                                size_t workspace_bytes, void* stream) {
  clear_error();
  ATTN_REQUIRE(q && k && lse && weights_out, "attn_key_weights: null pointer argument");
  ATTN_REQUIRE(dtype == ATTN_F32 || dtype == ATTN_BF16 || dtype == ATTN_TF32, "attn_key_weights: bad dtype");
  ATTN_REQUIRE(B > 0 && NH > 0 && NKV > 0 && T > 0 && D > 0, "attn_key_weights: sizes must be positive");
  ATTN_REQUIRE(NH % NKV == 0, "attn_key_weights: %d query heads are no multiple of %d key heads", NH, NKV);
  ATTN_REQUIRE(first_query >= 0, "attn_key_weights: first_query must not be negative");
  ATTN_REQUIRE(q_sb >= 0 && q_st >= 0 && q_sh >= 0 && k_sb >= 0 && k_st >= 0 && k_sh >= 0 && w_sb >= 0 && w_sh >= 0,
               "attn_key_weights: strides must not be negative");
  const RowSet w(T, B, w_sb, NKV, w_sh);
  ATTN_REQUIRE(w.apart, "attn_key_weights: rows of the weights must not overlap");
  ATTN_REQUIRE(!weights_in || weights_in == weights_out || !w.meets(weights_in, w, weights_out, 4),
               "attn_key_weights: weights_in and weights_out must be the same array or not overlap");
  const size_t esz = dtype == ATTN_BF16 ? 2 : 4;
  ATTN_REQUIRE(aligned(q, esz) && aligned(k, esz) && aligned(lse, 4), "attn_key_weights: misaligned tensor");
  if (D > 128) {
    set_error("attn_key_weights: head_dim %d not supported (up to 128)", D);
    return ATTN_ERR_UNSUPPORTED;
  }
  ATTN_REQUIRE(T <= 1 << 30, "attn_key_weights: T = %d exceeds 2^30", T);  // rows are ints with room to round up
  if ((int64_t)B * NKV * ((T + KW_TILE - 1) / KW_TILE) >= (int64_t)1 << 30) {
    set_error("attn_key_weights: too many key tiles for one launch; split the batch into several calls");
    return ATTN_ERR_UNSUPPORTED;
  }
  const KeyWeights p = {q, k, lse, weights_in, weights_out, q_sb, q_st, q_sh, k_sb, k_st, k_sh, w_sb, w_sh,
                        NH, NKV, NH / NKV, T, D, first_query, lengths, scale * 1.4426950408889634f};
  const size_t need = attn_key_weights_workspace_size(B, NKV, T);
  if (need && (!workspace || workspace_bytes < need)) {
    set_error("attn_key_weights: workspace of %zu bytes required", need);
    return ATTN_ERR_WORKSPACE;
  }
  ATTN_REQUIRE(aligned(workspace, 4), "attn_key_weights: misaligned workspace");
  if (key_weights_tc_ok(p, dtype)) return key_weights_tc(p, B, dtype == ATTN_TF32, (float*)workspace, as_stream(stream));
  return key_weights_simt(p, B, dtype, (float*)workspace, as_stream(stream));
}
