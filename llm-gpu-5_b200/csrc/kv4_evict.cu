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
// The select kernel finds the keep-th largest order key by radix (four passes of 8 bits over a
// histogram in shared memory), numbers the ties, holes and spare rows with block scans in slot order,
// and writes slots[i] = the row that slot i holds afterwards (-1 past the kept ones).  The move kernel
// copies rows.
#include "kv4.cuh"
#include <math.h>

namespace attn {

constexpr int EV_THREADS = 1024;
constexpr int EV_MOVE_THREADS = 256;

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
};

// Order of a row: larger is kept longer.  Protected rows first; then the weight by value (NaN last).
__device__ __forceinline__ uint32_t evict_key(const Kv4Evict& p, int64_t row_w, int j, int64_t protect_from) {
  const int64_t at = p.pos ? (int64_t)p.pos[row_w + j] : j;
  if (at >= protect_from) return 0xffffffffu;
  const float w = p.w[row_w + j] + 0.f;  // -0 counts as 0
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
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
    int y = red[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, off);
      if (lane >= off) y += z;
    }
    red[lane] = y;
  }
  __syncthreads();
  *total = red[31];
  return x - v + (warp ? red[warp - 1] : 0);
}

__global__ void __launch_bounds__(EV_THREADS) kv4_evict_select_kernel(const Kv4Evict p) {
  __shared__ uint32_t hist[256];
  __shared__ int red[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  grid_dependency_wait();
  grid_dependents_launch();
  const int bh = blockIdx.x, b = bh / p.NH, h = bh % p.NH;
  const int n = seq_length(p.lengths, b, p.L);
  int* slots = p.slots + (int64_t)bh * p.keep;
  if (n <= p.keep) {  // everything stays
    for (int i = threadIdx.x; i < p.keep; i += EV_THREADS) slots[i] = i < n ? i : -1;
    return;
  }
  const int64_t row_w = b * p.w_sb + h * p.w_sh;
  const int64_t protect_from = seq_value(p.seen, b, p.seen0) - p.recent;
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
    for (int j = threadIdx.x; j < n; j += EV_THREADS) {
      const uint32_t key = evict_key(p, row_w, j, protect_from);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int left = s_left, digit = 255;
      while (digit > 0 && (int)hist[digit] < left) left -= (int)hist[digit--];
      s_left = left;
      s_prefix = prefix | (uint32_t)digit << shift;
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
    const int rank = tie0 + block_scan(tie, red, &total);
    tie0 += total;
    const bool kept = j < n && (key > limit || (tie && rank < ties));
    const bool hole = j < p.keep && !kept, extra = j >= p.keep && kept;
    const int both = block_scan(hole | (int)extra << 16, red, &total);
    if (hole) holes[hole0 + (both & 0xffff)] = j;
    if (extra) spare[spare0 + (both >> 16)] = j;
    if (j < p.keep && kept) slots[j] = j;
    hole0 += total & 0xffff;
    spare0 += total >> 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < hole0; i += EV_THREADS) slots[holes[i]] = spare[i];
}

template <int D>
__global__ void __launch_bounds__(EV_MOVE_THREADS) kv4_evict_move_kernel(const Kv4Evict p) {
  // a row's codes go in words of 4 bytes: D / 8 threads a row, K in grid.z = 0, V in 1
  constexpr int LPR = D / 8, ROWS = EV_MOVE_THREADS / LPR;
  grid_dependency_wait();
  grid_dependents_launch();
  const int chunks = (p.keep + ROWS - 1) / ROWS;
  const int bh = blockIdx.x / chunks, i = (blockIdx.x % chunks) * ROWS + threadIdx.x / LPR, sub = threadIdx.x % LPR;
  if (i >= p.keep) return;
  const int from = p.slots[(int64_t)bh * p.keep + i];
  if (from < 0 || (p.in_place && from == i)) return;
  const int b = bh / p.NH, h = bh % p.NH;
  const int64_t s = blockIdx.y * p.src.si + b * p.src.sb + h * p.src.sh + from;
  const int64_t d = blockIdx.y * p.dst.si + b * p.dst.sb + h * p.dst.sh + i;
  *reinterpret_cast<uint32_t*>(p.dst.codes + d * (D / 2) + sub * 4) =
      *reinterpret_cast<const uint32_t*>(p.src.codes + s * (D / 2) + sub * 4);
  if (sub < kv4_groups(D)) p.dst.params[d * kv4_groups(D) + sub] = p.src.params[s * kv4_groups(D) + sub];
  if (blockIdx.y == 0 && sub == 0) {
    const int64_t ws = b * p.w_sb + h * p.w_sh + from, wd = b * p.dw_sb + h * p.dw_sh + i;
    p.dw[wd] = p.w[ws];
    if (p.dpos) p.dpos[wd] = p.pos ? p.pos[ws] : from;
  }
}

template <int D>
static cudaError_t kv4_evict_move(const Kv4Evict& p, int B, cudaStream_t s) {
  constexpr int ROWS = EV_MOVE_THREADS / (D / 8);
  const unsigned chunks = (p.keep + ROWS - 1) / ROWS;
  return launch_pdl(kv4_evict_move_kernel<D>, dim3(chunks * B * p.NH, 2), dim3(EV_MOVE_THREADS), 0, s, p);
}

}  // namespace attn

using namespace attn;

extern "C" size_t attn_kv4_evict_workspace_size(int B, int NH, int L, int keep) {
  if (B <= 0 || NH <= 0 || L <= 0 || keep <= 0) return 0;
  return (size_t)B * NH * 2 * keep * sizeof(int);
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
  ATTN_REQUIRE(in_place || (dst_codes != codes && dst_params != params && dst_weights != weights),
               "attn_kv4_evict: the destination must be another cache (NULL: in place)");
  ATTN_REQUIRE(c_si >= capacity && (B == 1 || c_sb >= capacity) && p.dst.si >= p.dst.cap && (B == 1 || p.dst.sb >= p.dst.cap),
               "attn_kv4_evict: cache rows must not overlap");
  ATTN_REQUIRE(w_sb >= 0 && w_sh >= 0 && dw_sb >= 0 && dw_sh >= 0, "attn_kv4_evict: strides must not be negative");
  ATTN_REQUIRE(L > 0 && L <= capacity, "attn_kv4_evict: length %d outside 1 .. capacity %d", L, capacity);
  ATTN_REQUIRE(keep > 0 && keep <= p.dst.cap, "attn_kv4_evict: keep %d outside 1 .. capacity %d", keep, p.dst.cap);
  ATTN_REQUIRE(recent >= 0 && recent <= keep, "attn_kv4_evict: recent %d outside 0 .. keep %d", recent, keep);
  ATTN_REQUIRE(weights && slots && (in_place || dst_weights), "attn_kv4_evict: null pointer argument");
  const size_t need = attn_kv4_evict_workspace_size(B, NH, L, keep);
  if (!workspace || workspace_bytes < need) {
    set_error("attn_kv4_evict: workspace of %zu bytes required", need);
    return ATTN_ERR_WORKSPACE;
  }
  ATTN_REQUIRE(aligned(workspace, 4), "attn_kv4_evict: misaligned workspace");
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
  cudaError_t e = launch_pdl(kv4_evict_select_kernel, dim3(B * NH), dim3(EV_THREADS), 0, s, p);
  count_launch();
  if (int rc = check_launch("kv4_evict_select_kernel", e)) return rc;
  switch (D) {
    case 16: e = kv4_evict_move<16>(p, B, s); break;
    case 32: e = kv4_evict_move<32>(p, B, s); break;
    case 64: e = kv4_evict_move<64>(p, B, s); break;
    default: e = kv4_evict_move<128>(p, B, s); break;
  }
  count_launch();
  return check_launch("kv4_evict_move_kernel", e);
}
