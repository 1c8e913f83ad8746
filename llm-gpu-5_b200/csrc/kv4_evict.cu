// Eviction from the 4-bit cache by accumulated attention weight.
//
// Of the n = lengths[b] rows of every (sequence, head) the `keep` best stay: first the protected ones,
// whose token position is at least seen - recent, then those of the largest accumulated weight; among
// equals the lowest slot.  Attention over a cache does not depend on the order of its rows, so the
// kept rows are not closed up: those below slot `keep` stay where they are, and those from slot `keep`
// on fill, in order, the slots below it that were given up.  A row moves only from a slot >= keep to a
// slot < keep, so the move can run in place with every row in parallel, and evicting one row of a full
// cache moves one row.
//
// One CTA selects for one (sequence, head).  Up to 32,768 rows it holds every row's order key in registers,
// consecutive rows to a thread, and finds the keep-th largest bit by bit from the top: up to 32 counts, each a
// warp reduction, one barrier and a sum over the warps (no atomics, so the weights' skewed exponents cost
// nothing).  After about nine of them the undecided keys are few enough for one to a thread, and a count is a
// barrier (730 cycles a round before, 50 after).  Longer sequences take a radix search, four passes of 8 bits
// over a histogram in shared memory.  Ties, holes and spare rows are numbered with block scans in slot order, and
// slots[i] = the row that slot i holds afterwards (-1 past the kept ones).  The rows are then copied, codes in
// 16-byte pieces: by the same CTA when there are few to move (one launch), else by a second kernel.  Measured for
// half of 32 x 8 heads of 8,192 rows of 64: select 19 us (a third of it loading the weights, a third counting), move
// 34 us (150 MB, 71 % of DRAM's rate: half of the rows come from scattered places); one of 513 rows of 12 heads:
// 8 us in one launch.
#include "attn_tc_common.cuh"
#include "kv4.cuh"
#include <math.h>
#include <type_traits>

namespace attn {

constexpr int EV_THREADS = 512;
constexpr int EV_WARPS = EV_THREADS / 32;
constexpr int EV_MOVE_THREADS = 256;
constexpr int EV_MOST = 64;  // rows per thread of the register select
constexpr int EV_SHARED = 32;  // up to here its lists are in shared memory, beyond in the workspace

struct Kv4Evict {
  Kv4View src, dst;
  const float* w;
  const int* pos;  // NULL: a row's position is its slot
  float* dw;
  int* dpos;
  int64_t w_sb, w_sh, dw_sb, dw_sh;
  int NH, L, keep, recent;
  const int* lengths;
  const int* seen;
  int seen0;
  int* slots;  // [B*NH][keep]
  int* spare;  // workspace [B*NH][2][keep]: holes, then the rows that fill them
  int in_place;
  int fused;   // the select kernel moves the rows too
};

// Order of a row: larger is kept longer.  Protected rows first; then the weight by value (NaN last).
__device__ __forceinline__ uint32_t evict_key(float weight, int64_t position, int64_t protect_from) {
  if (position >= protect_from) return 0xffffffffu;
  const float w = weight + 0.f;  // -0 counts as 0
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint32_t evict_key(const Kv4Evict& p, int64_t row_w, int j, int64_t protect_from) {
  return evict_key(p.w[row_w + j], p.pos ? (int64_t)p.pos[row_w + j] : j, protect_from);
}

// Exclusive prefix of v over the block, and its total.
__device__ __forceinline__ int block_scan(int v, int* red, int* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int x = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int y = lane < EV_WARPS ? red[lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, off);
      if (lane >= off) y += z;
    }
    if (lane < EV_WARPS) red[lane] = y;
  }
  __syncthreads();
  *total = red[EV_WARPS - 1];
  return x - v + (warp ? red[warp - 1] : 0);
}

// Sum over the block of a value that is already summed over each warp (lane 0's counts).
__device__ __forceinline__ int block_total(int warp_total, int* red) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (lane == 0) red[warp] = warp_total;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, lane < EV_WARPS ? red[lane] : 0);
}

// Copy rows [first, first + count) of the kept ones of one (sequence, head): slot i gets row slots[i].
template <int D>
__device__ __forceinline__ void evict_move(const Kv4Evict& p, int b, int h, const int* slots, int first, int count) {
  constexpr int GROUPS = kv4_groups(D);
  using Unit = typename std::conditional<(D >= 32), uint4, uint2>::type;
  constexpr int UNITS = D / 2 / sizeof(Unit);  // of a row's codes
  constexpr int BATCH = 4;                     // loads in flight per thread
  const int64_t s0 = b * p.src.sb + h * p.src.sh, d0 = b * p.dst.sb + h * p.dst.sh;
  const int64_t ws = b * p.w_sb + h * p.w_sh, wd = b * p.dw_sb + h * p.dw_sh;
  for (int i = first + threadIdx.x; i < first + count; i += blockDim.x) {
    const int from = slots[i];
    if (from < 0 || (p.in_place && from == i)) continue;
    __half2 k[GROUPS], v[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      k[g] = p.src.params[(s0 + from) * GROUPS + g];
      v[g] = p.src.params[(p.src.si + s0 + from) * GROUPS + g];
    }
    const float w = p.w[ws + from];
    const int at = p.pos ? p.pos[ws + from] : from;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      p.dst.params[(d0 + i) * GROUPS + g] = k[g];
      p.dst.params[(p.dst.si + d0 + i) * GROUPS + g] = v[g];
    }
    p.dw[wd + i] = w;
    if (p.dpos) p.dpos[wd + i] = at;
  }
  // keys' units, then values', in one sequence: a chunk of 256 rows is one batch for 256 threads
  const Unit* src = reinterpret_cast<const Unit*>(p.src.codes) + s0 * UNITS;
  Unit* dst = reinterpret_cast<Unit*>(p.dst.codes) + (d0 + first) * UNITS;
  const int units = count * UNITS;
  for (int u0 = threadIdx.x; u0 < 2 * units; u0 += blockDim.x * BATCH) {
    Unit x[BATCH];
    bool go[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int v = u0 + k * blockDim.x, u = v < units ? v : v - units, i = first + u / UNITS;
      const int from = v < 2 * units ? slots[i] : -1;
      go[k] = from >= 0 && !(p.in_place && from == i);
      if (go[k]) x[k] = src[((v < units ? 0 : p.src.si) + from) * UNITS + u % UNITS];
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int v = u0 + k * blockDim.x, u = v < units ? v : v - units;
      if (go[k]) dst[(v < units ? 0 : p.dst.si) * UNITS + u] = x[k];
    }
  }
}

// PER rows per thread in registers; PER = 0: any number of rows, read again for every pass.
template <int D, int PER>
__global__ void __launch_bounds__(EV_THREADS) kv4_evict_select_kernel(const Kv4Evict p) {
  __shared__ int red[2][EV_WARPS];
  grid_dependency_wait();
  grid_dependents_launch();
  const int bh = blockIdx.x, b = bh / p.NH, h = bh % p.NH;
  const int n = seq_length(p.lengths, b, p.L);
  int* slots = p.slots + (int64_t)bh * p.keep;
  if (n <= p.keep) {  // everything stays
    for (int i = threadIdx.x; i < p.keep; i += EV_THREADS) slots[i] = i < n ? i : -1;
  } else {
    const int64_t row_w = b * p.w_sb + h * p.w_sh;
    const int64_t protect_from = seq_value(p.seen, b, p.seen0) - p.recent;
    if constexpr (PER > 0) {
      const int base = threadIdx.x * PER;
      // at most min(keep, n - keep) each
      constexpr int LIST = PER <= EV_SHARED ? EV_THREADS * PER / 2 : 1;
      __shared__ uint16_t s_holes[LIST], s_spare[LIST];
      uint16_t* holes = PER <= EV_SHARED ? s_holes : reinterpret_cast<uint16_t*>(p.spare + (int64_t)bh * 2 * p.keep);
      uint16_t* spare = PER <= EV_SHARED ? s_spare : holes + p.keep;
      uint32_t key[PER];
      const bool wide = PER % 4 == 0 && row_w % 4 == 0 && (reinterpret_cast<uintptr_t>(p.w) | reinterpret_cast<uintptr_t>(p.pos)) % 16 == 0;
      if (wide && base + PER <= n) {
#pragma unroll
        for (int k = 0; k < PER; k += 4) {
          const float4 w = *reinterpret_cast<const float4*>(p.w + row_w + base + k);
          const int4 at = p.pos ? *reinterpret_cast<const int4*>(p.pos + row_w + base + k)
                                : make_int4(base + k, base + k + 1, base + k + 2, base + k + 3);
          key[k] = evict_key(w.x, at.x, protect_from);
          if constexpr (PER % 4 == 0) {
            key[k + 1] = evict_key(w.y, at.y, protect_from);
            key[k + 2] = evict_key(w.z, at.z, protect_from);
            key[k + 3] = evict_key(w.w, at.w, protect_from);
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < PER; ++k) key[k] = base + k < n ? evict_key(p, row_w, base + k, protect_from) : 0u;
      }
      // count(key >= limit) = lo >= keep, and count(key >= limit + bit) = hi < keep.  Rows past the end have key
      // 0, which no candidate counts.
      __shared__ uint32_t list[EV_THREADS];
      uint32_t limit = 0, bit = 0x80000000u;
      int lo = n, hi = 0, round = 0;
      for (; bit && lo != p.keep && lo - hi > EV_THREADS; bit >>= 1, ++round) {
        const uint32_t cand = limit | bit;
        int c = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k)  // c += key >= cand, as the carry of key - cand: two instructions a key
          asm("{\n\t.reg .u32 t;\n\tadd.cc.u32 t, %1, %2;\n\taddc.u32 %0, %0, 0;\n\t}" : "+r"(c) : "r"(key[k]), "r"(0u - cand));
        const int total = block_total(__reduce_add_sync(0xffffffffu, c), red[round & 1]);
        if (total >= p.keep) {
          limit = cand;
          lo = total;
        } else {
          hi = total;
        }
      }
      // (lo == keep: these are the kept ones, and no lower bit can change that)
      if (bit && lo != p.keep) {
        // no more undecided keys than threads: a thread takes one, and a round is a counting barrier
        const uint32_t last = limit + (bit - 1) + bit;
        int in = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) in += base + k < n && key[k] >= limit && key[k] <= last;
        int all;
        int at = block_scan(in, red[round & 1], &all);
#pragma unroll
        for (int k = 0; k < PER; ++k)
          if (base + k < n && key[k] >= limit && key[k] <= last) list[at++] = key[k];
        __syncthreads();
        const uint32_t mine = threadIdx.x < all ? list[threadIdx.x] : 0u;
        const int need = p.keep - hi;
        for (; bit; bit >>= 1) {
          const int total = __syncthreads_count(mine >= (limit | bit));
          if (total >= need) limit |= bit;
          if (total == need) break;
        }
      }
      int above = 0, tie = 0;
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        above += key[k] > limit;
        tie += base + k < n && key[k] == limit;
      }
      __syncthreads();  // (either half of red may have been read last)
      const int ties = p.keep - block_total(__reduce_add_sync(0xffffffffu, above), red[0]);
      int total;
      int rank = block_scan(tie, red[1], &total);
      typename std::conditional<(PER <= 32), uint32_t, uint64_t>::type kept = 0;
      int count = 0;  // holes, and spare rows in the upper half
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int j = base + k;
        const bool same = j < n && key[k] == limit;
        const bool stay = j < n && (key[k] > limit || (same && rank < ties));
        rank += same;
        kept |= (decltype(kept))stay << k;
        if (j < n && j < p.keep && !stay) count += 1;
        if (j >= p.keep && stay) count += 1 << 16;
      }
      // every slot keeps its row, in one coalesced sweep; the holes are written over below
      for (int i = threadIdx.x; i < p.keep; i += EV_THREADS) slots[i] = i;
      int at = block_scan(count, red[0], &total);
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int j = base + k;
        const bool stay = (kept >> k & 1) != 0;
        if (j < p.keep) {
          if (!stay && j < n) {
            holes[at & 0xffff] = (uint16_t)j;
            at += 1;
          }
        } else if (stay) {
          spare[at >> 16] = (uint16_t)j;
          at += 1 << 16;
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < (total & 0xffff); i += EV_THREADS) slots[holes[i]] = spare[i];
    } else {
      __shared__ uint32_t hist[256];
      __shared__ uint32_t s_prefix;
      __shared__ int s_left;
      // the keep-th largest key, digit by digit from the top; s_left = how many of the rows that match
      // the prefix so far are still to be kept
      if (threadIdx.x == 0) {
        s_prefix = 0;
        s_left = p.keep;
      }
      for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) hist[threadIdx.x] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix, mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
        for (int j0 = 0; j0 < n; j0 += EV_THREADS) {
          const int j = j0 + threadIdx.x;
          const uint32_t key = j < n ? evict_key(p, row_w, j, protect_from) : 0u;
          const uint32_t digit = j < n && (key & mask) == prefix ? (key >> shift) & 255u : 256u;
          // lanes of one digit (weights share few exponents) add as one
          const uint32_t peers = __match_any_sync(0xffffffffu, digit);
          if (digit < 256u && threadIdx.x % 32 == __ffs(peers) - 1) atomicAdd(&hist[digit], __popc(peers));
        }
        __syncthreads();
        if (threadIdx.x < 32) {  // lane l: digits 255 - 8 l downwards
          const int lane = threadIdx.x;
          int c[8], sum = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) sum += c[k] = (int)hist[255 - 8 * lane - k];
          int before = sum;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, before, off);
            if (lane >= off) before += y;
          }
          before -= sum;
          const int left = s_left;
          __syncwarp();
          if (before < left && before + sum >= left) {  // exactly one lane
            int k = 0;
            while (k < 7 && before + c[k] < left) before += c[k++];
            s_left = left - before;
            s_prefix = prefix | (uint32_t)(255 - 8 * lane - k) << shift;
          }
        }
        __syncthreads();
      }
      const uint32_t limit = s_prefix;
      const int ties = s_left;  // rows equal to the limit that are kept, the lowest slots first
      int* holes = p.spare + (int64_t)bh * 2 * p.keep;
      int* spare = holes + p.keep;
      int tie0 = 0, hole0 = 0, spare0 = 0;
      for (int base = 0; base < n; base += EV_THREADS) {
        const int j = base + threadIdx.x;
        const uint32_t key = j < n ? evict_key(p, row_w, j, protect_from) : 0u;
        const bool tie = j < n && key == limit;
        int total;
        const int rank = tie0 + block_scan(tie, red[0], &total);
        tie0 += total;
        const bool kept = j < n && (key > limit || (tie && rank < ties));
        const bool hole = j < p.keep && !kept, extra = j >= p.keep && kept;
        const int both = block_scan(hole | (int)extra << 16, red[1], &total);
        if (hole) holes[hole0 + (both & 0xffff)] = j;
        if (extra) spare[spare0 + (both >> 16)] = j;
        if (j < p.keep && kept) slots[j] = j;
        hole0 += total & 0xffff;
        spare0 += total >> 16;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < hole0; i += EV_THREADS) slots[holes[i]] = spare[i];
    }
  }
  if (p.fused) {
    __syncthreads();
    evict_move<D>(p, b, h, slots, 0, min(n, p.keep));
  }
}

template <int D>
__global__ void __launch_bounds__(EV_MOVE_THREADS) kv4_evict_move_kernel(const Kv4Evict p) {
  grid_dependency_wait();
  grid_dependents_launch();
  const int chunks = (p.keep + EV_MOVE_THREADS - 1) / EV_MOVE_THREADS;
  const int bh = blockIdx.x / chunks, first = (blockIdx.x - bh * chunks) * EV_MOVE_THREADS;
  const int b = bh / p.NH, h = bh - b * p.NH;
  evict_move<D>(p, b, h, p.slots + (int64_t)bh * p.keep, first, min(EV_MOVE_THREADS, p.keep - first));
}

template <int D>
static int kv4_evict_d(Kv4Evict& p, int B, cudaStream_t s) {
  // one launch where there is little to move and few slots to look through.  Measured, in one and in two, one row out
  // of 8 heads of 1,025 rows 8.0 and 8.4 us, of 2,049 10.4 and 9.6, of 4,096 17.0 and 12.5, of 8,192 27.8 and 17.2; out of
  // 128 heads 8.2 and 10.2, 10.8 and 14.2, 17.6 and 17.4, 28.7 and 27.8; out of 256 heads 14.3 and 15.0, 15.2 and 16.9,
  // 26.5 and 28.0, 45.6 and 47.6 (there the CTAs fill the GPU either way); half of 256 heads of 2,000 rows 17.1 and 17.4,
  // of 8,192 59.6 and 55.5
  const int rows = p.in_place ? (p.L - p.keep < p.keep ? p.L - p.keep : p.keep) : (p.L < p.keep ? p.L : p.keep);
  const int64_t heads = (int64_t)B * p.NH;
  p.fused = rows <= 1024 && p.keep <= 2048;
  const dim3 grid((unsigned)heads), block(EV_THREADS);
  cudaError_t e;
  // the fewest rows per thread that hold the sequence: idle threads and wide loops both cost (256 heads of 4,000 rows:
  // 18 us with 16 a thread, of 10,330 rows 40 us with 32; one row
  // out of 8 heads of 32,000: 70 us with 64, 209 with the passes over memory)
  if (p.L <= EV_THREADS) e = launch_pdl(kv4_evict_select_kernel<D, 1>, grid, block, 0, s, p);
  else if (p.L <= 4 * EV_THREADS) e = launch_pdl(kv4_evict_select_kernel<D, 4>, grid, block, 0, s, p);
  else if (p.L <= 8 * EV_THREADS) e = launch_pdl(kv4_evict_select_kernel<D, 8>, grid, block, 0, s, p);
  else if (p.L <= 16 * EV_THREADS) e = launch_pdl(kv4_evict_select_kernel<D, 16>, grid, block, 0, s, p);
  else if (p.L <= EV_SHARED * EV_THREADS) e = launch_pdl(kv4_evict_select_kernel<D, EV_SHARED>, grid, block, 0, s, p);
  else if (p.L <= EV_MOST * EV_THREADS) e = launch_pdl(kv4_evict_select_kernel<D, EV_MOST>, grid, block, 0, s, p);
  else e = launch_pdl(kv4_evict_select_kernel<D, 0>, grid, block, 0, s, p);
  count_launch();
  if (int rc = check_launch("kv4_evict_select_kernel", e)) return rc;
  if (p.fused) return ATTN_OK;
  const unsigned chunks = (p.keep + EV_MOVE_THREADS - 1) / EV_MOVE_THREADS;
  e = launch_pdl(kv4_evict_move_kernel<D>, dim3(chunks * (unsigned)heads), dim3(EV_MOVE_THREADS), 0, s, p);
  count_launch();
  return check_launch("kv4_evict_move_kernel", e);
}

}  // namespace attn

using namespace attn;

extern "C" size_t attn_kv4_evict_workspace_size(int B, int NH, int L, int keep) {
  if (B <= 0 || NH <= 0 || L <= 0 || keep <= 0) return 0;
  return L <= attn::EV_SHARED * attn::EV_THREADS ? 0 : (size_t)B * NH * 2 * keep * sizeof(int);
}

extern "C" int attn_kv4_evict(void* codes, void* params, float* weights, int* positions, int64_t c_si, int64_t c_sb,
                              int64_t c_sh, int capacity, int64_t w_sb, int64_t w_sh, void* dst_codes, void* dst_params,
                              float* dst_weights, int* dst_positions, int64_t d_si, int64_t d_sb, int64_t d_sh,
                              int dst_capacity, int64_t dw_sb, int64_t dw_sh, int B, int NH, int L, int D, int keep,
                              int recent, const int* lengths, const int* seen, int seen0, int* slots, void* workspace,
                              size_t workspace_bytes, void* stream) {
  clear_error();
  const bool in_place = dst_codes == nullptr;
  Kv4Evict p = {};
  p.src = {(uint8_t*)codes, (__half2*)params, c_si, c_sb, c_sh, capacity};
  p.dst = in_place ? p.src : Kv4View{(uint8_t*)dst_codes, (__half2*)dst_params, d_si, d_sb, d_sh, dst_capacity};
  if (int rc = kv4_check("attn_kv4_evict", p.src, B, NH, D)) return rc;
  if (int rc = kv4_check("attn_kv4_evict", p.dst, B, NH, D)) return rc;
  ATTN_REQUIRE(RowSet(capacity, 2, c_si, B, c_sb, NH, c_sh).apart &&
                   RowSet(p.dst.cap, 2, p.dst.si, B, p.dst.sb, NH, p.dst.sh).apart,
               "attn_kv4_evict: cache rows must not overlap");
  ATTN_REQUIRE(w_sb >= 0 && w_sh >= 0 && dw_sb >= 0 && dw_sh >= 0, "attn_kv4_evict: strides must not be negative");
  ATTN_REQUIRE(L > 0 && L <= capacity, "attn_kv4_evict: length %d outside 1 .. capacity %d", L, capacity);
  ATTN_REQUIRE(keep > 0 && keep <= p.dst.cap, "attn_kv4_evict: keep %d outside 1 .. capacity %d", keep, p.dst.cap);
  ATTN_REQUIRE(recent >= 0 && recent <= keep, "attn_kv4_evict: recent %d outside 0 .. keep %d", recent, keep);
  ATTN_REQUIRE(weights && slots && (in_place || dst_weights), "attn_kv4_evict: null pointer argument");
  if (!in_place) {
    const RowSet rows(L, 2, c_si, B, c_sb, NH, c_sh), kept(keep, 2, d_si, B, d_sb, NH, d_sh);
    ATTN_REQUIRE(!kept.meets(dst_codes, rows, codes, D / 2) && !kept.meets(dst_params, rows, params, 4 * kv4_groups(D)),
                 "attn_kv4_evict: the destination must be another cache (NULL: in place)");
  }
  const size_t need = attn_kv4_evict_workspace_size(B, NH, L, keep);
  if (need && (!workspace || workspace_bytes < need)) {
    set_error("attn_kv4_evict: workspace of %zu bytes required", need);
    return ATTN_ERR_WORKSPACE;
  }
  ATTN_REQUIRE(aligned(workspace, 4), "attn_kv4_evict: misaligned workspace");
  const RowSet w(L, B, w_sb, NH, w_sh);
  ATTN_REQUIRE(w.apart, "attn_kv4_evict: rows of the weights must not overlap");
  if (!in_place) {
    const RowSet kept(keep, B, dw_sb, NH, dw_sh);
    ATTN_REQUIRE(kept.apart, "attn_kv4_evict: rows of the weights must not overlap");
    ATTN_REQUIRE(!kept.meets(dst_weights, w, weights, 4) && !(positions && dst_positions && kept.meets(dst_positions, w, positions, 4)),
                 "attn_kv4_evict: the destination must be another cache (NULL: in place)");
  }
  if ((int64_t)B * NH * ((keep + 15) / 16) >= (int64_t)1 << 31) {
    set_error("attn_kv4_evict: B*NH*keep = %lld rows are too many for one call; split the batch", (long long)B * NH * keep);
    return ATTN_ERR_UNSUPPORTED;
  }
  p.w = weights; p.pos = positions; p.dw = in_place ? weights : dst_weights;
  p.dpos = in_place ? positions : dst_positions;
  p.w_sb = w_sb; p.w_sh = w_sh; p.dw_sb = in_place ? w_sb : dw_sb; p.dw_sh = in_place ? w_sh : dw_sh;
  p.NH = NH; p.L = L; p.keep = keep; p.recent = recent;
  p.lengths = lengths; p.seen = seen; p.seen0 = seen0;
  p.slots = slots; p.spare = (int*)workspace; p.in_place = in_place;
  cudaStream_t s = as_stream(stream);
  switch (D) {
    case 16: return kv4_evict_d<16>(p, B, s);
    case 32: return kv4_evict_d<32>(p, B, s);
    case 64: return kv4_evict_d<64>(p, B, s);
    default: return kv4_evict_d<128>(p, B, s);
  }
}
