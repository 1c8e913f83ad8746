// Quantise keys and values into the 4-bit cache (store) and read rows back as numbers (load).
//
// The reference has no key/value cache (generate.py:611-628 runs the whole context again for every
// token); these fill and read the one attn_kv4_decode attends over.  Both are one pass: the store
// reads each value once and writes 4 bits and 1/16 of a scale pair for it, so HBM traffic bounds the
// prompt's store and launch latency a single token's.
//
// A row is taken by D / 8 lanes of 8 values each (16 bytes of bf16 per lane); a group's minimum and
// maximum come from shuffles among its 2, 4 or 8 lanes.  Rows are walked in runs of up to a CTA's rows of
// one head, all heads of those positions in turn: a warp's codes (and scale pairs) of consecutive
// positions are one contiguous write, its reads whole rows of the token layout, and the heads that share
// a token's DRAM page are read at about the same time.  A thread takes the key and the value of its
// place, so that the index arithmetic is shared by 16 values.  Measured for 32 x 1,024 tokens of 8 heads of 64 in
// bfloat16: store 36 us (67 MB read, 19 written; 21 us with the quantisation left out, so its instructions are
// the bound), load 18.5 us (86 MB, 4.7 TB/s).
#include "kv4.cuh"
#include <math.h>

namespace attn {

constexpr int KV4_THREADS = 256;

int kv4_check(const char* fn, const Kv4View& c, int B, int NH, int D) {
  ATTN_REQUIRE(c.codes && c.params, "%s: null cache pointer", fn);
  ATTN_REQUIRE(B > 0 && NH > 0 && c.cap > 0, "%s: B, NH and capacity must be positive", fn);
  if (!kv4_head_dim_ok(D)) {
    set_error("%s: head_dim %d not supported by the 4-bit cache (16, 32, 64 or 128)", fn, D);
    return ATTN_ERR_UNSUPPORTED;
  }
  ATTN_REQUIRE(c.cap % KV4_ALIGN_ROWS == 0 && c.si % KV4_ALIGN_ROWS == 0 && c.sb % KV4_ALIGN_ROWS == 0 &&
                   c.sh % KV4_ALIGN_ROWS == 0,
               "%s: the cache's capacity and strides must be multiples of %d rows", fn, KV4_ALIGN_ROWS);
  ATTN_REQUIRE(c.cap <= 1 << 30, "%s: capacity %d exceeds 2^30 rows", fn, c.cap);  // positions are ints with room to round up
  ATTN_REQUIRE(c.si >= 0 && c.sb >= 0 && c.sh >= c.cap, "%s: bad cache strides", fn);
  ATTN_REQUIRE(aligned(c.codes, 16) && aligned(c.params, 16), "%s: the cache must be 16-byte aligned", fn);
  return ATTN_OK;
}

struct Kv4Rows {
  const void *k, *v;
  int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  uint32_t T, NH;
  uint32_t rows, run;  // row = ((b * runs + position / run) * NH + h) * run + position % run; rows with padding
  FastDiv by_run, by_nh, by_runs;
};

// Positions per run (`most`: the rows of a CTA), and the number of rows with the last run of every
// sequence filled up.
static inline int64_t kv4_set_rows(Kv4Rows* r, int B, uint32_t most) {
  r->run = r->T < most ? r->T : most;
  const uint32_t runs = (r->T + r->run - 1) / r->run;
  const int64_t rows = (int64_t)B * runs * r->NH * r->run;
  r->rows = (uint32_t)rows;
  r->by_run.set(r->run);
  r->by_nh.set(r->NH);
  r->by_runs.set(runs);
  return rows;
}

// The row of a thread.  WHOLE: a CTA is one run, so all but the position is the same for its threads
// and stays in uniform registers.
template <int LPR, bool WHOLE>
struct Kv4Row {
  uint32_t b, h, t;
  bool in;
  __device__ __forceinline__ explicit Kv4Row(const Kv4Rows& a) {
    constexpr uint32_t PER = KV4_THREADS / LPR;
    uint32_t q, place = threadIdx.x / LPR;
    in = true;
    if constexpr (WHOLE) {
      q = blockIdx.x;
    } else {
      const uint32_t row = blockIdx.x * PER + place;
      in = row < a.rows;
      q = a.by_run.div(min(row, a.rows - 1));
      place = min(row, a.rows - 1) - q * a.run;
    }
    const uint32_t u = a.by_nh.div(q);
    h = q - u * a.NH;
    b = a.by_runs.div(u);
    t = (u - b * a.by_runs.d) * a.run + place;
    in = in && t < a.T;
  }
};

struct Kv4Slots {
  const int* starts;  // first slot of each sequence: starts[b] + start
  int start;
  const int* counts;  // tokens of each sequence (NULL: T)
};

struct Kv4Marks {
  float* weights;  // zeroed at the stored slots (may be NULL)
  int* positions;  // token positions, seen[b] + seen0 + t (may be NULL)
  int64_t sb, sh;
  const int* seen;
  int seen0;
};

// Eight values, and their smallest and largest.  hi is +infinity where one of them is not finite.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&x)[8], float& lo, float& hi) {
  if constexpr (VEC && sizeof(T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);  // two at a time
    const __nv_bfloat162 mn = __hmin2(__hmin2(h[0], h[1]), __hmin2(h[2], h[3]));
    const __nv_bfloat162 mx = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    lo = fminf(__low2float(mn), __high2float(mn));
    hi = fmaxf(__low2float(mx), __high2float(mx));
  } else {
    if constexpr (VEC) {
      const float4 a = load4(p), b = load4(p + 4);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = Elem<T>::load(p + i);
    }
    lo = hi = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
    }
  }
  float zero = 0.f;  // stays 0 while everything is finite
#pragma unroll
  for (int i = 0; i < 8; ++i) zero = __fmaf_rn(x[i], 0.f, zero);
  if (!(zero == 0.f)) hi = INFINITY;
}

template <typename T, int D, bool VEC, bool WHOLE>
__global__ void __launch_bounds__(KV4_THREADS)
kv4_store_kernel(const Kv4Rows in, const Kv4View c, const Kv4Slots sl, const Kv4Marks mk) {
  constexpr int LPR = D / 8;             // lanes per row
  constexpr int LPG = kv4_group(D) / 8;  // lanes per group
  grid_dependency_wait();
  grid_dependents_launch();
  const int sub = threadIdx.x % LPR;
  const Kv4Row<LPR, WHOLE> at(in);
  const uint32_t b = at.b, h = at.h, t = at.t;
  const int64_t slot = seq_value(sl.starts, b, sl.start) + t;
  const bool put = at.in && slot >= 0 && slot < c.cap && (int64_t)t < seq_value(sl.counts, b, sl.counts ? 0 : in.T);
  const int64_t dst0 = b * c.sb + h * c.sh + slot;
  float x[2][8], lo[2] = {0.f, 0.f}, hi[2] = {0.f, 0.f};
  if (put) {
    load8<T, VEC>((const T*)in.k + b * in.k_sb + t * in.k_st + h * in.k_sh + sub * 8, x[0], lo[0], hi[0]);
    load8<T, VEC>((const T*)in.v + b * in.v_sb + t * in.v_st + h * in.v_sh + sub * 8, x[1], lo[1], hi[1]);
  }
#pragma unroll
  for (int off = LPG / 2; off > 0; off >>= 1)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      lo[i] = fminf(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], off));
      hi[i] = fmaxf(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], off));
    }
  if (!put) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // scale and minimum saturate at float16's largest value; a group holding an infinity or a NaN reads
    // back as NaN
    const bool fin = hi[i] < INFINITY;
    const __half s = __float2half_rn(fin ? fminf(__fmul_rn(__fsub_rn(hi[i], lo[i]), 1.f / 15.f), 65504.f) : NAN);
    const __half m = __float2half_rn(fin ? fminf(fmaxf(lo[i], -65504.f), 65504.f) : NAN);
    const float sf = __half2float(s);
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(sf));  // (unused where s is 0 or NaN)
    const uint32_t w = kv4_word(x[i], sf, __half2float(m), inv);
    const int64_t dst = dst0 + i * c.si;
    *reinterpret_cast<uint32_t*>(c.codes + dst * (D / 2) + sub * 4) = w;
    if (sub % LPG == 0) c.params[dst * kv4_groups(D) + sub / LPG] = __halves2half2(s, m);
  }
  if (sub == 0 && (mk.weights || mk.positions)) {
    const int64_t mark = b * mk.sb + h * mk.sh + slot;
    if (mk.weights) mk.weights[mark] = 0.f;
    if (mk.positions) mk.positions[mark] = (int)(seq_value(mk.seen, b, mk.seen0) + t);
  }
}

template <typename T, int D, bool VEC, bool WHOLE>
__global__ void __launch_bounds__(KV4_THREADS)
kv4_load_kernel(const Kv4Rows out, const Kv4View c, const Kv4Slots sl) {
  constexpr int LPR = D / 8;
  constexpr int LPG = kv4_group(D) / 8;
  grid_dependency_wait();
  grid_dependents_launch();
  const int sub = threadIdx.x % LPR;
  const Kv4Row<LPR, WHOLE> at(out);
  if (!at.in) return;
  const uint32_t b = at.b, h = at.h, t = at.t;
  const int64_t slot = seq_value(sl.starts, b, sl.start) + t;
  const bool held = slot >= 0 && slot < c.cap && (int64_t)t < seq_value(sl.counts, b, sl.counts ? 0 : out.T);
  const int64_t src = b * c.sb + h * c.sh + slot, to = b * out.k_sb + t * out.k_st + h * out.k_sh + sub * 8;
  uint32_t w[2] = {0, 0};
  float2 p[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};  // reads as zeros
  if (held)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = *reinterpret_cast<const uint32_t*>(c.codes + (src + i * c.si) * (D / 2) + sub * 4);
      p[i] = __half22float2(c.params[(src + i * c.si) * kv4_groups(D) + sub / LPG]);
    }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float x[8];
    kv4_values(w[i], p[i].x, p[i].y, x);
    T* dst = (T*)(i ? out.v : out.k) + to;
    if constexpr (VEC && sizeof(T) == 2) {
      uint32_t w2[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
        w2[k] = *reinterpret_cast<const uint32_t*>(&v);
      }
      *reinterpret_cast<uint4*>(dst) = make_uint4(w2[0], w2[1], w2[2], w2[3]);
    } else if constexpr (VEC) {
      store4(dst, make_float4(x[0], x[1], x[2], x[3]));
      store4(dst + 4, make_float4(x[4], x[5], x[6], x[7]));
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) Elem<T>::store(dst + k, x[k]);
    }
  }
}

template <typename T, int D, bool VEC, bool WHOLE>
static cudaError_t kv4_rows_start(const Kv4Rows& r, const Kv4View& c, const Kv4Slots& sl, const Kv4Marks* mk, cudaStream_t s) {
  constexpr uint32_t per = KV4_THREADS / (D / 8);
  const dim3 grid((r.rows + per - 1) / per);
  return mk ? launch_pdl(kv4_store_kernel<T, D, VEC, WHOLE>, grid, dim3(KV4_THREADS), 0, s, r, c, sl, *mk)
            : launch_pdl(kv4_load_kernel<T, D, VEC, WHOLE>, grid, dim3(KV4_THREADS), 0, s, r, c, sl);
}

template <typename T, int D, bool VEC>
static int kv4_rows_launch(const Kv4Rows& r, const Kv4View& c, const Kv4Slots& sl, const Kv4Marks* mk, cudaStream_t s) {
  // sequences of at least a CTA's rows take CTAs of their own; the rows of shorter ones share them
  const cudaError_t e = r.run == KV4_THREADS / (D / 8) ? kv4_rows_start<T, D, VEC, true>(r, c, sl, mk, s)
                                                      : kv4_rows_start<T, D, VEC, false>(r, c, sl, mk, s);
  count_launch();
  return check_launch(mk ? "kv4_store_kernel" : "kv4_load_kernel", e);
}

template <typename T>
static int kv4_rows_t(const Kv4Rows& r, int D, const Kv4View& c, const Kv4Slots& sl, const Kv4Marks* mk, cudaStream_t s) {
  // 16-byte accesses where every lane's first value is aligned for them
  constexpr int64_t V = 16 / sizeof(T);
  const bool vec = aligned(r.k, 16) && aligned(r.v, 16) && r.k_sb % V == 0 && r.k_st % V == 0 && r.k_sh % V == 0 &&
                   r.v_sb % V == 0 && r.v_st % V == 0 && r.v_sh % V == 0;
#define KV4_ROWS(DD)                                                       \
  case DD:                                                                 \
    return vec ? kv4_rows_launch<T, DD, true>(r, c, sl, mk, s) : kv4_rows_launch<T, DD, false>(r, c, sl, mk, s);
  switch (D) { KV4_ROWS(16) KV4_ROWS(32) KV4_ROWS(64) KV4_ROWS(128) }
#undef KV4_ROWS
  return ATTN_ERR_UNSUPPORTED;
}

static int kv4_rows(const char* fn, Kv4Rows r, int B, int D, int dtype, const Kv4View& c, const Kv4Slots& sl,
                    const Kv4Marks* mk, cudaStream_t s) {
  ATTN_REQUIRE(r.k && r.v, "%s: null pointer argument", fn);
  ATTN_REQUIRE(dtype == ATTN_F32 || dtype == ATTN_BF16, "%s: dtype must be ATTN_F32 or ATTN_BF16", fn);
  ATTN_REQUIRE(aligned(r.k, dtype == ATTN_BF16 ? 2 : 4) && aligned(r.v, dtype == ATTN_BF16 ? 2 : 4), "%s: misaligned tensor", fn);
  const int64_t st[6] = {r.k_sb, r.k_st, r.k_sh, r.v_sb, r.v_st, r.v_sh};
  for (int i = 0; i < 6; ++i) ATTN_REQUIRE(st[i] >= 0, "%s: strides must not be negative", fn);
  ATTN_REQUIRE(sl.starts || (sl.start >= 0 && (int64_t)sl.start + r.T <= c.cap),
               "%s: positions %d .. %lld exceed the capacity of %d", fn, sl.start, (long long)sl.start + r.T - 1, c.cap);
  if (!mk) {  // what the load writes
    const RowSet o(D, B, r.k_sb, r.T, r.k_st, r.NH, r.k_sh);
    ATTN_REQUIRE(o.apart && !o.meets(r.k, o, r.v, dtype == ATTN_BF16 ? 2 : 4), "%s: rows of the output must not overlap", fn);
  }
  ATTN_REQUIRE(kv4_set_rows(&r, B, KV4_THREADS / (D / 8)) < (int64_t)1 << 31, "%s: B*NH*T must be below 2^31", fn);
  return dtype == ATTN_BF16 ? kv4_rows_t<__nv_bfloat16>(r, D, c, sl, mk, s) : kv4_rows_t<float>(r, D, c, sl, mk, s);
}

}  // namespace attn

using namespace attn;

extern "C" int attn_kv4_store(const void* k, const void* v, int dtype, int B, int T, int NH, int D, int64_t k_sb,
                              int64_t k_st, int64_t k_sh, int64_t v_sb, int64_t v_st, int64_t v_sh, void* codes,
                              void* params, int64_t c_si, int64_t c_sb, int64_t c_sh, int capacity, const int* starts,
                              int start, const int* counts, float* weights, int* positions, int64_t w_sb, int64_t w_sh,
                              const int* seen, int seen0, void* stream) {
  clear_error();
  ATTN_REQUIRE(B > 0 && T > 0 && NH > 0, "attn_kv4_store: sizes must be positive");
  ATTN_REQUIRE((int64_t)B * NH * T < (int64_t)1 << 31, "attn_kv4_store: B*NH*T must be below 2^31");
  ATTN_REQUIRE(!(weights || positions) || (w_sb >= 0 && w_sh >= 0), "attn_kv4_store: bad strides");
  const Kv4Rows r = {k, v, k_sb, k_st, k_sh, v_sb, v_st, v_sh, (uint32_t)T, (uint32_t)NH};
  const Kv4View c = {(uint8_t*)codes, (__half2*)params, c_si, c_sb, c_sh, capacity};
  if (int rc = kv4_check("attn_kv4_store", c, B, NH, D)) return rc;
  ATTN_REQUIRE(RowSet(capacity, 2, c_si, B, c_sb, NH, c_sh).apart, "attn_kv4_store: cache rows must not overlap");
  ATTN_REQUIRE(!(weights || positions) || RowSet(capacity, B, w_sb, NH, w_sh).apart,
               "attn_kv4_store: rows of weights and positions must not overlap");
  const Kv4Marks mk = {weights, positions, w_sb, w_sh, seen, seen0};
  return kv4_rows("attn_kv4_store", r, B, D, dtype, c, Kv4Slots{starts, start, counts}, &mk, as_stream(stream));
}

extern "C" int attn_kv4_load(const void* codes, const void* params, int64_t c_si, int64_t c_sb, int64_t c_sh,
                             int capacity, int B, int T, int NH, int D, const int* starts, int start, const int* counts,
                             void* k, void* v, int dtype, int64_t o_sb, int64_t o_st, int64_t o_sh, void* stream) {
  clear_error();
  ATTN_REQUIRE(B > 0 && T > 0 && NH > 0, "attn_kv4_load: sizes must be positive");
  ATTN_REQUIRE((int64_t)B * NH * T < (int64_t)1 << 31, "attn_kv4_load: B*NH*T must be below 2^31");
  const Kv4Rows r = {k, v, o_sb, o_st, o_sh, o_sb, o_st, o_sh, (uint32_t)T, (uint32_t)NH};
  const Kv4View c = {(uint8_t*)codes, (__half2*)params, c_si, c_sb, c_sh, capacity};
  if (int rc = kv4_check("attn_kv4_load", c, B, NH, D)) return rc;
  return kv4_rows("attn_kv4_load", r, B, D, dtype, c, Kv4Slots{starts, start, counts}, nullptr, as_stream(stream));
}
