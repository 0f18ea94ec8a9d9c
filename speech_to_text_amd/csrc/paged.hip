// Paged K/V cache: block tables and slot maps from request lengths, and attention of drafted token
// trees over the cache (stt_paged_plan, stt_tree_attention of include/stt_mi355x.h).
#include "stt_common.h"

typedef uint16_t half_bits;

namespace {

// ---------------------------------------------------------------------------------------------
// Plan of one step.  need_i = ceil((cached_i + new_i) / P), take_i = max(0, need_i - held_i),
// give_i = max(0, held_i - need_i); the exclusive sums of take, give and new over the requests say
// which ring entries and rows a request gets.  Every block repeats the scan (8 192 requests are
// 96 KB of lengths out of the L2) and then serves its own share of the requests, a group of
// `group` lanes each, so one launch does without a grid-wide step between scan and fill.
// Ring entries taken (head ..) and returned (tail ..) are disjoint modulo the ring's size (checked),
// and a request's table row is touched by its own lane group only.
// ---------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

struct PlanArgs {
  const int32_t *cached, *fresh;
  int n, shift;
  int32_t* table;
  int width;
  int32_t* free_ids;
  int n_ring;
  const int64_t* ring_in;
  int64_t* ring_out;
  const int32_t* held_in;
  int32_t* held_out;
  int rows;
  int32_t* starts;
  int64_t* slots;
  int32_t* positions;
  int32_t* status;
  int group;            // lanes per request, a power of two <= 64
};

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(const PlanArgs a) {
  __shared__ int32_t s_take[STT_PLAN_MAX_REQUESTS], s_give[STT_PLAN_MAX_REQUESTS], s_start[STT_PLAN_MAX_REQUESTS];
  __shared__ long long wave_sum[3][kPlanThreads / 64];
  __shared__ int wave_bad[kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long head = a.ring_in[0], tail = a.ring_in[1];
  const int per = (a.n + kPlanThreads - 1) / kPlanThreads;

  // blocks to take and return and new rows of request i; false (and zeros) if it is malformed
  auto demand = [&](int i, int& take, int& give, int& fresh, int& bad) __attribute__((always_inline)) {
    take = give = fresh = 0;
    const int c = a.cached[i], w = a.fresh[i], h = a.held_in[i];
    const long long need = ((long long)c + w + ((1LL << a.shift) - 1)) >> a.shift;
    if (c < 0 || w < 0 || h < 0 || h > a.width) bad |= 1;
    else if (need > a.width) bad |= 2;
    else {
      const int d = (int)need - h;
      take = d > 0 ? d : 0;
      give = d < 0 ? -d : 0;
      fresh = w;
    }
  };
  // this thread's run of consecutive requests
  long long own[3] = {0, 0, 0};
  int bad = 0;                                 // bit 0: bad state, bit 1: too long
  for (int i = tid * per; i < tid * per + per && i < a.n; ++i) {
    int take, give, fresh;
    demand(i, take, give, fresh, bad);
    own[0] += take; own[1] += give; own[2] += fresh;
  }
  // exclusive scan over the threads: inside the wave, then over the waves
  long long before[3];
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    long long v = own[q];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const long long up = __shfl_up(v, o, 64);
      if (lane >= o) v += up;
    }
    if (lane == 63) wave_sum[q][wave] = v;
    before[q] = v - own[q];
  }
  const int any = __any(bad & 1) ? 1 : 0, any2 = __any(bad & 2) ? 2 : 0;
  if (lane == 0) wave_bad[wave] = any | any2;
  __syncthreads();
  long long total[3] = {0, 0, 0};
  int wrong = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      if (w < wave) before[q] += wave_sum[q][w];
      total[q] += wave_sum[q][w];
    }
    wrong |= wave_bad[w];
  }
  int status = STT_PLAN_OK;
  if ((wrong & 1) || head < 0 || tail < head || tail - head > a.n_ring || tail + total[1] - head > a.n_ring)
    status = STT_PLAN_BAD_STATE;
  else if (wrong & 2) status = STT_PLAN_TOO_LONG;
  else if (total[0] > tail - head) status = STT_PLAN_NO_BLOCKS;
  else if (total[2] > a.rows) status = STT_PLAN_TOO_MANY_ROWS;
  const long first = (long)blockIdx.x * kPlanThreads + tid, stride = (long)gridDim.x * kPlanThreads;
  if (first == 0) {
    a.status[0] = status;
    a.ring_out[0] = status ? head : head + total[0];
    a.ring_out[1] = status ? tail : tail + total[1];
    a.starts[a.n] = status ? 0 : (int)total[2];
  }
  if (status) {                                // uniform over the grid: nothing changes, nothing to do
    for (long i = first; i < a.n; i += stride) { a.held_out[i] = a.held_in[i]; a.starts[i] = 0; }
    for (long r = first; r < a.rows; r += stride) { a.slots[r] = -1; a.positions[r] = -1; }
    return;
  }
  for (int i = tid * per; i < tid * per + per && i < a.n; ++i) {
    int take, give, fresh;
    demand(i, take, give, fresh, bad);
    s_take[i] = (int)before[0]; s_give[i] = (int)before[1]; s_start[i] = (int)before[2];
    before[0] += take; before[1] += give; before[2] += fresh;
  }
  __syncthreads();
  for (long r = total[2] + first; r < a.rows; r += stride) { a.slots[r] = -1; a.positions[r] = -1; }

  const int hm = (int)(head % a.n_ring), tm = (int)(tail % a.n_ring);
  const int sub = tid & (a.group - 1);
  const long groups = stride / a.group;
  for (long g = first / a.group; g < a.n; g += groups) {
    const int i = (int)g;
    const int c = a.cached[i], w = a.fresh[i], h = a.held_in[i];
    const int need = (int)(((long long)c + w + ((1LL << a.shift) - 1)) >> a.shift);
    const int t0 = s_take[i], g0 = s_give[i], r0 = s_start[i];
    int32_t* row = a.table + (long)i * a.width;
    if (sub == 0) { a.held_out[i] = need; a.starts[i] = r0; }
    for (int j = sub; j < w; j += a.group) {
      const int pos = c + j, b = pos >> a.shift;
      int id;
      if (b < h) id = row[b];
      else {
        long at = (long)hm + t0 + (b - h);
        id = a.free_ids[at >= a.n_ring ? at - a.n_ring : at];
      }
      a.positions[r0 + j] = pos;
      a.slots[r0 + j] = ((long long)id << a.shift) + (pos & ((1 << a.shift) - 1));
    }
    for (int j = sub; j < need - h; j += a.group) {
      const long at = (long)hm + t0 + j;
      row[h + j] = a.free_ids[at >= a.n_ring ? at - a.n_ring : at];
    }
    for (int j = sub; j < h - need; j += a.group) {
      const long at = (long)tm + g0 + j;
      a.free_ids[at >= a.n_ring ? at - a.n_ring : at] = row[need + j];
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Tree attention.  A block owns one (sequence, KV head), a slice of its keys and a tile of query
// rows; row r of the (sequence, KV head) is node r / group, query head r % group of the group.
// Keys come in tiles of 32: cached positions, then (last slice) the tree's own nodes, whose K/V the
// block also stores into the cache.  Per tile, S^T = K Q^T and O^T += V^T P^T on the matrix cores
// (v_mfma_f32_16x16x32): a lane holds one query against 8 keys, so maximum, sum and rescale factor
// are per lane; the two score products of a tile take the keys 8a + b and 8a + 4 + b (a, b < 4), so
// that the exponentiated scores of lane group g are the keys 8g .. 8g + 7 in order and, rounded to
// the storage type, already are the B operand of the second product.  K and V go through LDS images
// (rows padded by 16 bytes) as they come from memory; V is read back transposed.
//   The softmax keeps a reference r <= max <= r + 8 per query (base-2 units): it is moved, and the sums
// rescaled, only when a tile raises the maximum more than 8 above it, so weights are at most 2^8.
//   WR = 1: each of the four waves walks its own tiles (every fourth) for all 16 NR rows of the block,
// staging through wave-private images without barriers, and the waves' (reference, sum, O) are joined
// at the end: few rows, memory bound.  WR = 4: the waves share each tile and own 16 NR rows each.
// ---------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(4))) float pa_f4;
typedef __attribute__((ext_vector_type(4))) uint32_t pa_u4;
typedef __attribute__((ext_vector_type(2))) uint32_t pa_u2;
typedef __attribute__((ext_vector_type(4))) short pa_s4;
typedef __attribute__((ext_vector_type(8))) __bf16 pa_b8;
typedef __attribute__((ext_vector_type(8))) _Float16 pa_h8;
typedef __attribute__((ext_vector_type(2))) __bf16 pa_b2;
typedef __attribute__((ext_vector_type(2))) _Float16 pa_h2;
typedef __attribute__((ext_vector_type(2))) float pa_f2;

template <typename T> struct Half;
template <> struct Half<__bf16> {
  static __device__ __forceinline__ float up(half_bits v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(pa_f2{a, b}, pa_b2)); }
  static __device__ __forceinline__ pa_f4 mfma(pa_u4 a, pa_u4 b, pa_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_b8, a), __builtin_bit_cast(pa_b8, b), c, 0, 0, 0);
  }
  static constexpr uint32_t kExponent = 0x7F80, kOne = 0x3F80, kMinusMark = 0x4300, kNanMark = 0x4680;   // 1, 128, 16384
};
template <> struct Half<_Float16> {
  static __device__ __forceinline__ float up(half_bits v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(pa_f2{a, b}, pa_h2)); }
  static __device__ __forceinline__ pa_f4 mfma(pa_u4 a, pa_u4 b, pa_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pa_h8, a), __builtin_bit_cast(pa_h8, b), c, 0, 0, 0);
  }
  static constexpr uint32_t kExponent = 0x7C00, kOne = 0x3C00, kMinusMark = 0x5800, kNanMark = 0x7400;
};

// Path of each node of one tree as a 64-bit set, by pointer jumping: after s rounds a node's set holds
// its nearest 2^s ancestors.  Lane l computes node l; parents outside [0, own index) are roots.
__device__ __forceinline__ unsigned long long tree_path(const int32_t* parents, int row0, int nodes, int lane) {
  int up = -1;
  if (lane < nodes) {
    up = parents ? parents[row0 + lane] : lane - 1;
    if (up >= lane) up = -1;
  }
  unsigned long long seen = 1ull << lane;
#pragma unroll
  for (int s = 0; s < 6; ++s) {
    const int src = up < 0 ? lane : up;
    const unsigned long long more = __shfl(seen, src, 64);
    const int next = __shfl(up, src, 64);
    if (up >= 0) { seen |= more; up = next; }
  }
  return seen;
}

struct TreeShape {
  int chunk;        // cached positions per slice, a multiple of 32
  int slices;       // slices in the grid; a sequence uses ceil(cached / chunk) of them, at least one
  int row_tiles;    // blocks per (sequence, KV head, slice)
  float* part;      // [rows][heads][slices][D] unnormalised sums of the slices, and
  float* stat;      // [rows][heads][slices][2] their (reference, sum); unused with one slice
};

// cached positions of a sequence as far as its table reaches
__device__ __forceinline__ int tree_history(const stt_tree_attention_args& a, int seq) {
  const int c = a.d_cached[seq];
  const long most = a.n_blocks > 0 ? (long)a.width * a.block_size : 0;
  return c < 0 ? 0 : c < most ? c : (int)most;
}
__device__ __forceinline__ int tree_slices(int cached, const TreeShape& sh) {
  if (sh.slices == 1 || cached <= sh.chunk) return 1;
  const int n = (cached + sh.chunk - 1) / sh.chunk;
  return n < sh.slices ? n : sh.slices;             // the last one takes whatever is left
}

constexpr int kTile = 32;

// One wave's queries and running sums, and the work on one 32-key tile.
template <typename T, int D, int NR>
struct TreeWave {
  static constexpr int kPitch = D * 2 + 16;          // bytes per key row of an image
  static constexpr int kImage = kTile * kPitch;
  pa_u4 q[NR][D / 32];
  pa_f4 o[NR][D / 16];
  float ref[NR], sum[NR];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int x = 0; x < NR; ++x) {
      ref[x] = -__builtin_inff();
      sum[x] = 0.f;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) o[x][t] = pa_f4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // two stored values without their infinities and NaNs; `count` receives what those count as
  static __device__ __forceinline__ uint32_t split(uint32_t u, uint32_t& count) {
    uint32_t out = 0;
    count = 0;
#pragma unroll
    for (int b = 0; b < 32; b += 16) {
      const uint32_t h = (u >> b) & 0xFFFFu, e = Half<T>::kExponent;
      if ((h & e) != e) out |= h << b;
      else count |= (uint32_t)((h & 0x7FFFu) != e ? Half<T>::kNanMark : h >> 15 ? Half<T>::kMinusMark : Half<T>::kOne) << b;
    }
    return out;
  }
  // 1.0 for each of the two lowest bits that is set
  static __device__ __forceinline__ uint32_t ones(uint32_t bits) {
    return (bits & 1 ? Half<T>::kOne : 0u) | (bits & 2 ? Half<T>::kOne << 16 : 0u);
  }

  // keep[x]: bit j set: the lane's query x sees key 8 g + j of the tile (looked at if `masked`).
  // spoiled: some value of the tile is not finite and may belong to a key a query does not see; a zero
  // weight would still turn it into NaN on the matrix cores.  Then the finite values are multiplied
  // alone, a second product counts the infinities and NaNs among the keys a query does see (exact
  // small integers: +inf 1, -inf 128, NaN 16384, at most 32 keys), and those are added afterwards.
  __device__ __forceinline__ void tile(const unsigned char* kimg, const unsigned char* vimg, const uint32_t (&keep)[NR],
                                       bool masked, bool spoiled, float scale2, int lane) {
    const int col = lane & 15, g = lane >> 4;
    const unsigned char* ka = kimg + (8 * (col >> 2) + (col & 3)) * kPitch + 16 * g;
    pa_f4 s1[NR], s2[NR];
#pragma unroll
    for (int x = 0; x < NR; ++x) s1[x] = s2[x] = pa_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const pa_u4 a0 = *(const pa_u4*)(ka + 64 * c), a1 = *(const pa_u4*)(ka + 4 * kPitch + 64 * c);
#pragma unroll
      for (int x = 0; x < NR; ++x) {
        s1[x] = Half<T>::mfma(a0, q[x][c], s1[x]);
        s2[x] = Half<T>::mfma(a1, q[x][c], s2[x]);
      }
    }
    pa_u4 pf[NR];
    float p[NR][8];
#pragma unroll
    for (int x = 0; x < NR; ++x) {
#pragma unroll
      for (int r = 0; r < 4; ++r) { p[x][r] = s1[x][r] * scale2; p[x][4 + r] = s2[x][r] * scale2; }
      if (masked) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[x][j] = (keep[x] >> j) & 1 ? p[x][j] : -__builtin_inff();
      }
      float top = fmaxf(fmaxf(fmaxf(p[x][0], p[x][1]), fmaxf(p[x][2], p[x][3])), fmaxf(fmaxf(p[x][4], p[x][5]), fmaxf(p[x][6], p[x][7])));
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any(top > ref[x] + 8.0f)) {
        // (both -inf: nothing seen yet, the sums are zero whatever the factor)
        const float next = top > ref[x] + 8.0f ? top : ref[x];
        const float f = next == ref[x] ? 1.0f : __builtin_amdgcn_exp2f(ref[x] - next);
        ref[x] = next;
        sum[x] *= f;
#pragma unroll
        for (int t = 0; t < D / 16; ++t) o[x][t] *= f;
      }
      const float base = ref[x] == -__builtin_inff() ? 0.f : ref[x];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[x][j] = __builtin_amdgcn_exp2f(p[x][j] - base);
      sum[x] += ((p[x][0] + p[x][1]) + (p[x][2] + p[x][3])) + ((p[x][4] + p[x][5]) + (p[x][6] + p[x][7]));
      pf[x].x = Half<T>::pack(p[x][0], p[x][1]); pf[x].y = Half<T>::pack(p[x][2], p[x][3]);
      pf[x].z = Half<T>::pack(p[x][4], p[x][5]); pf[x].w = Half<T>::pack(p[x][6], p[x][7]);
    }
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      // transposed read: lane 4 u + w of a 16-lane group addresses key row 8 g + 4 half + u, features
      // 16 t + 4 w ..; lane i receives feature 16 t + i of the four keys
      const unsigned char* at = vimg + (8 * g + (col >> 2)) * kPitch + (16 * t + 4 * (col & 3)) * 2;
      const pa_u2 lo = __builtin_bit_cast(pa_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)at));
      const pa_u2 hi = __builtin_bit_cast(pa_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)(at + 4 * kPitch)));
      pa_u4 v = {lo.x, lo.y, hi.x, hi.y};
      if (spoiled) {
        uint32_t c0, c1, c2, c3;
        v = pa_u4{split(v.x, c0), split(v.y, c1), split(v.z, c2), split(v.w, c3)};
        const pa_u4 count = {c0, c1, c2, c3};
#pragma unroll
        for (int x = 0; x < NR; ++x) {
          pa_u4 sees;
          sees.x = ones(keep[x]); sees.y = ones(keep[x] >> 2); sees.z = ones(keep[x] >> 4); sees.w = ones(keep[x] >> 6);
          const pa_f4 c = Half<T>::mfma(count, sees, pa_f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int k = (int)c[r];
            if (k >> 14) o[x][t][r] = __builtin_nanf("");
            if (k & 127) o[x][t][r] += __builtin_inff();
            if ((k >> 7) & 127) o[x][t][r] -= __builtin_inff();
          }
        }
      }
#pragma unroll
      for (int x = 0; x < NR; ++x) o[x][t] = Half<T>::mfma(v, pf[x], o[x][t]);
    }
  }
};

// 16-byte pieces of one key tile as a group of LANES threads holds them: piece = key * (D / 8) + part
template <int D, int LANES>
struct TilePieces {
  static constexpr int kPer = kTile * (D / 8) / LANES;
  static constexpr int kKeysPerStep = LANES / (D / 8);
  pa_u4 k[kPer], v[kPer];
};

template <typename T, int D, int NR, int WR, bool WIDE>
__global__ __launch_bounds__(256, NR == 1 ? (D == 64 ? 3 : 2) : NR == 2 ? 2 : 1) void tree_attention_kernel(
    const stt_tree_attention_args a, const TreeShape sh) {
  typedef TreeWave<T, D, NR> Wave;
  constexpr int LANES = WR == 1 ? 64 : 256;          // threads that load a tile together
  typedef TilePieces<D, LANES> Pieces;
  __shared__ __attribute__((aligned(16))) unsigned char lds[WR == 1 ? 8 : 4][Wave::kImage];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int col = lane & 15, g = lane >> 4;
  long id = blockIdx.x;
  const int slice = (int)(id % sh.slices);
  id /= sh.slices;
  const int rt = (int)(id % sh.row_tiles);
  id /= sh.row_tiles;
  const int hk = (int)(id % a.n_kv_heads), seq = (int)(id / a.n_kv_heads);
  const int row0 = a.d_starts[seq];
  int nodes = a.d_starts[seq + 1] - row0;
  nodes = nodes < a.max_nodes ? nodes : a.max_nodes;
  if (nodes <= 0 || row0 < 0 || row0 > a.rows - nodes) return;
  const int group = a.n_heads / a.n_kv_heads, n_rows = nodes * group;
  const int first_row = rt * 16 * NR * WR;
  const int cached = tree_history(a, seq), used = tree_slices(cached, sh);
  if (first_row >= n_rows || slice >= used) return;
  const int key0 = slice * sh.chunk;
  const int key1 = slice == used - 1 ? cached : key0 + sh.chunk;
  const int hist_tiles = (key1 - key0 + kTile - 1) / kTile;
  const int tiles = hist_tiles + (slice == used - 1 ? (nodes + kTile - 1) / kTile : 0);
  const int shift = __builtin_ctz(a.block_size);

  Wave w;
  w.clear();
  const int wave_row = first_row + (WR == 1 ? 0 : wave * 16 * NR);
  int node[NR];
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    int r = wave_row + 16 * x + col;
    r = r < n_rows ? r : n_rows - 1;
    node[x] = r / group;
    const half_bits* q = (const half_bits*)a.d_q + (row0 + node[x]) * a.q_row + (hk * group + (r - node[x] * group)) * a.q_head + 8 * g;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) w.q[x][c] = *(const pa_u4*)(q + 32 * c);
  }
  const float scale2 = a.scale * 1.4426950408889634f;

  const half_bits* kc = (const half_bits*)a.d_k_cache + hk * a.head_stride;
  const half_bits* vc = (const half_bits*)a.d_v_cache + hk * a.head_stride;
  const int loader = WR == 1 ? lane : tid;
  const int piece = loader % (D / 8), key_in = loader / (D / 8);

  // Block ids of a tile's positions.  WIDE (blocks of 32 positions and more): the tile lies in one block.
  // Otherwise lane l holds the id of the tile's position l (l < 32); -1 where there is none.
  auto load_ids = [&](int t) __attribute__((always_inline)) -> int {
    if (t >= hist_tiles) return -1;
    const int at = (key0 + t * kTile + (WIDE ? 0 : (lane & 31))) >> shift;
    return at < a.width ? a.d_table[(long)seq * a.width + at] : -1;
  };
  // positions of the tile that exist and have a block, as a bit set
  auto valid = [&](int t, int ids) __attribute__((always_inline)) -> uint32_t {
    const bool ok = key0 + t * kTile + (lane & 31) < key1 && (uint32_t)ids < (uint32_t)a.n_blocks;
    return (uint32_t)__ballot(ok);
  };
  auto load = [&](int t, int ids, Pieces& p) __attribute__((always_inline)) {
    if (t < hist_tiles) {
      const int pos = key0 + t * kTile;
      const int use = (uint32_t)ids < (uint32_t)a.n_blocks ? ids : 0;
      if (WIDE) {
        const long base = __builtin_amdgcn_readfirstlane(use) * a.block_stride + (pos & (a.block_size - 1)) * a.pos_stride;
        const uint32_t off = (uint32_t)(key_in * (int)a.pos_stride + 8 * piece);
#pragma unroll
        for (int i = 0; i < Pieces::kPer; ++i) {
          const long at = base + (long)i * Pieces::kKeysPerStep * a.pos_stride;
          p.k[i] = *(const pa_u4*)(kc + at + off);
          p.v[i] = *(const pa_u4*)(vc + at + off);
        }
      } else {
#pragma unroll
        for (int i = 0; i < Pieces::kPer; ++i) {
          const int key = key_in + i * Pieces::kKeysPerStep;
          const int b = __shfl(use, key, 64);
          const long at = b * a.block_stride + ((pos + key) & (a.block_size - 1)) * a.pos_stride + 8 * piece;
          p.k[i] = *(const pa_u4*)(kc + at);
          p.v[i] = *(const pa_u4*)(vc + at);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < Pieces::kPer; ++i) {
        int nd = (t - hist_tiles) * kTile + key_in + i * Pieces::kKeysPerStep;
        nd = nd < nodes ? nd : nodes - 1;
        p.k[i] = *(const pa_u4*)((const half_bits*)a.d_k + (long)(row0 + nd) * a.k_row + hk * a.k_head + 8 * piece);
        p.v[i] = *(const pa_u4*)((const half_bits*)a.d_v + (long)(row0 + nd) * a.v_row + hk * a.v_head + 8 * piece);
      }
    }
  };
  // registers -> LDS images; values of positions that do not exist become zero
  auto stage = [&](Pieces& p, uint32_t ok, unsigned char* kimg, unsigned char* vimg) __attribute__((always_inline)) {
    if (ok != 0xFFFFFFFFu) {
#pragma unroll
      for (int i = 0; i < Pieces::kPer; ++i)
        if (!((ok >> (key_in + i * Pieces::kKeysPerStep)) & 1)) p.v[i] = pa_u4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < Pieces::kPer; ++i) {
      const int at = (key_in + i * Pieces::kKeysPerStep) * Wave::kPitch + 16 * piece;
      *(pa_u4*)(kimg + at) = p.k[i];
      *(pa_u4*)(vimg + at) = p.v[i];
    }
  };
  // a tree tile: the nodes' K/V into the cache (one row tile does it); is some value not finite?
  auto store_nodes = [&](int t, const Pieces& p) __attribute__((always_inline)) -> bool {
    bool odd = false;
#pragma unroll
    for (int i = 0; i < Pieces::kPer; ++i) {
      const int nd = (t - hist_tiles) * kTile + key_in + i * Pieces::kKeysPerStep;
      const uint32_t e = Half<T>::kExponent, u[4] = {p.v[i].x, p.v[i].y, p.v[i].z, p.v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) odd |= (u[j] & e) == e || (u[j] & (e << 16)) == (e << 16);
      if (rt == 0 && nd < nodes) {
        const long slot = a.d_slots[row0 + nd];
        if (slot >= 0 && slot < ((long)a.n_blocks << shift)) {
          const long at = (slot >> shift) * a.block_stride + hk * a.head_stride + (slot & (a.block_size - 1)) * a.pos_stride + 8 * piece;
          *(pa_u4*)((half_bits*)a.d_k_cache + at) = p.k[i];
          *(pa_u4*)((half_bits*)a.d_v_cache + at) = p.v[i];
        }
      }
    }
    return odd;
  };
  unsigned long long path = 0;                       // of node `lane`
  if (tiles > hist_tiles) path = tree_path(a.d_parents, row0, nodes, lane);
  auto compute = [&](int t, uint32_t ok, bool spoiled, const unsigned char* kimg, const unsigned char* vimg) __attribute__((always_inline)) {
    uint32_t keep[NR];
    const bool tree = t >= hist_tiles;
#pragma unroll
    for (int x = 0; x < NR; ++x) keep[x] = (ok >> (8 * g)) & 255u;
    if (tree) {
#pragma unroll
      for (int x = 0; x < NR; ++x) keep[x] = (uint32_t)(__shfl(path, node[x], 64) >> ((t - hist_tiles) * kTile + 8 * g)) & 255u;
    }
    w.tile(kimg, vimg, keep, tree || ok != 0xFFFFFFFFu, spoiled, scale2, lane);
  };

  if (WR == 1) {
    unsigned char *kimg = lds[2 * wave], *vimg = lds[2 * wave + 1];
    // Two register sets alternate between "in flight" and "being used"; block ids are fetched one
    // tile further ahead, since the addresses of the next loads wait for them.
    Pieces pa, pb;
    int ia = load_ids(wave), ib = load_ids(wave + 4);
    if (wave < tiles) load(wave, ia, pa);
    auto run = [&](int t, int ids, Pieces& p) __attribute__((always_inline)) {
      const bool tree = t >= hist_tiles;
      const int left = nodes - (t - hist_tiles) * kTile;
      const uint32_t ok = !tree ? valid(t, ids) : left >= kTile ? 0xFFFFFFFFu : (1u << left) - 1;
      bool spoiled = false;
      if (tree) spoiled = __any(store_nodes(t, p));
      stage(p, ok, kimg, vimg);
      compute(t, ok, spoiled, kimg, vimg);
    };
    for (int t = wave; t < tiles; t += 8) {
      const int ia2 = load_ids(t + 8), ib2 = load_ids(t + 12);
      if (t + 4 < tiles) load(t + 4, ib, pb);
      run(t, ia, pa);
      if (t + 8 < tiles) load(t + 8, ia2, pa);
      if (t + 4 < tiles) run(t + 4, ib, pb);
      ia = ia2; ib = ib2;
    }
  } else {
    // tile t in images (t & 1); while it is worked on the next one is on its way to registers
    Pieces p;
    int ids = load_ids(0);
    __shared__ int spoiled_flag[2];
    if (tid < 2) spoiled_flag[tid] = 0;
    __syncthreads();
    if (tiles > 0) load(0, ids, p);
    for (int t = 0; t < tiles; ++t) {              // stage tile t, then work on it behind the barrier
      const bool tree = t >= hist_tiles;
      const int left = nodes - (t - hist_tiles) * kTile;
      const uint32_t ok = !tree ? valid(t, ids) : left >= kTile ? 0xFFFFFFFFu : (1u << left) - 1;
      if (tree && store_nodes(t, p)) spoiled_flag[t & 1] = 1;
      stage(p, ok, lds[2 * (t & 1)], lds[2 * (t & 1) + 1]);
      const int next = load_ids(t + 1);
      __syncthreads();
      if (t + 1 < tiles) load(t + 1, next, p);
      compute(t, ok, tree && spoiled_flag[t & 1], lds[2 * (t & 1)], lds[2 * (t & 1) + 1]);
      ids = next;
    }
    __syncthreads();
  }

  // results.  A lane holds features 16 t + 4 g + r of query `col` of each sub-tile.
  auto write = [&](int r, float refv, float sumv, int feature, pa_f4 v) __attribute__((always_inline)) {
    const int nd = r / group, h = hk * group + (r - nd * group);
    if (used == 1) {
      const float inv = 1.0f / sumv;
      half_bits* out = (half_bits*)a.d_out + (row0 + nd) * a.out_row + h * a.out_head + feature;
      *(pa_u2*)out = pa_u2{Half<T>::pack(v[0] * inv, v[1] * inv), Half<T>::pack(v[2] * inv, v[3] * inv)};
    } else {
      const long at = ((long)(row0 + nd) * a.n_heads + h) * sh.slices + slice;
      *(pa_f4*)(sh.part + at * D + feature) = v;
      if (feature == 0) { sh.stat[2 * at] = refv; sh.stat[2 * at + 1] = sumv; }
    }
  };
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    float sum = w.sum[x];
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (WR == 4) {
      const int r = wave_row + 16 * x + col;
      if (r < n_rows) {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) write(r, w.ref[x], sum, 16 * t + 4 * g, w.o[x][t]);
      }
      continue;
    }
    // join the four waves: [query][feature] of each in its own images, then (reference, sum)
    float* mine = (float*)lds[2 * wave];
    constexpr int kRow = D + 4;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < D / 16; ++t) *(pa_f4*)(mine + col * kRow + 16 * t + 4 * g) = w.o[x][t];
    if (g == 0) { mine[16 * kRow + col] = w.ref[x]; mine[16 * kRow + 16 + col] = sum; }
    __syncthreads();
    for (int e = tid; e < 16 * (D / 4); e += 256) {
      const int qi = e / (D / 4), f = 4 * (e % (D / 4));
      const int r = first_row + 16 * x + qi;
      if (r >= n_rows) continue;
      float rf[4], top = -__builtin_inff();
#pragma unroll
      for (int u = 0; u < 4; ++u) { rf[u] = ((const float*)lds[2 * u])[16 * kRow + qi]; top = fmaxf(top, rf[u]); }
      pa_f4 num = {0.f, 0.f, 0.f, 0.f};
      float den = 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float* src = (const float*)lds[2 * u];
        const float f2 = rf[u] == -__builtin_inff() ? (src[16 * kRow + 16 + qi] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(rf[u] - top);
        if (f2 != 0.f) {
          num += f2 * *(const pa_f4*)(src + qi * kRow + f);
          den += f2 * src[16 * kRow + 16 + qi];
        }
      }
      write(r, top, den, f, num);
    }
  }
}

// Joins the slices of a (row, head) in slice order; thread = feature.
template <typename T, int D>
__global__ __launch_bounds__(D) void tree_join_kernel(const stt_tree_attention_args a, const TreeShape sh) {
  long id = blockIdx.x;
  const int h = (int)(id % a.n_heads);
  id /= a.n_heads;
  const int node = (int)(id % a.max_nodes), seq = (int)(id / a.max_nodes);
  const int row0 = a.d_starts[seq];
  int nodes = a.d_starts[seq + 1] - row0;
  nodes = nodes < a.max_nodes ? nodes : a.max_nodes;
  if (node >= nodes || row0 < 0 || row0 > a.rows - nodes) return;
  const int used = tree_slices(tree_history(a, seq), sh);
  if (used == 1) return;
  const long at = ((long)(row0 + node) * a.n_heads + h) * sh.slices;
  float top = -__builtin_inff();
  for (int s = 0; s < used; ++s) top = fmaxf(top, sh.stat[2 * (at + s)]);
  float num = 0.f, den = 0.f;
  for (int s = 0; s < used; ++s) {
    const float rf = sh.stat[2 * (at + s)], l = sh.stat[2 * (at + s) + 1];
    const float f = rf == -__builtin_inff() ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(rf - top);
    if (f != 0.f) {
      num += f * sh.part[(at + s) * D + threadIdx.x];
      den += f * l;
    }
  }
  ((half_bits*)a.d_out)[(row0 + node) * a.out_row + h * a.out_head + threadIdx.x] = (half_bits)Half<T>::pack(num / den, 0.f);
}

bool power_of_two(int v) { return v > 0 && (v & (v - 1)) == 0; }

// 0, or the error of a malformed argument block
int check_tree(const stt_tree_attention_args* a) {
  if (!a) return stt_fail(STT_ERR_INVALID_ARGUMENT, "null argument");
  if (a->n_seq < 0 || a->rows < 0 || a->n_heads < 1 || a->n_kv_heads < 1 || a->n_heads % a->n_kv_heads || a->n_blocks < 0 ||
      a->width < 0)
    return stt_fail(STT_ERR_INVALID_ARGUMENT, "bad sizes (%d sequences, %d rows, %d / %d heads, %d blocks, width %d)",
                    a->n_seq, a->rows, a->n_heads, a->n_kv_heads, a->n_blocks, a->width);
  if (a->head_dim != 64 && a->head_dim != 128) return stt_fail(STT_ERR_UNSUPPORTED, "head size %d: 64 or 128", a->head_dim);
  if (a->dtype != STT_BF16 && a->dtype != STT_F16) return stt_fail(STT_ERR_UNSUPPORTED, "dtype %d: STT_BF16 or STT_F16", a->dtype);
  if (!power_of_two(a->block_size) || a->block_size > 65536)
    return stt_fail(STT_ERR_UNSUPPORTED, "block size %d: a power of two <= 65536", a->block_size);
  if (a->max_nodes < 1 || a->max_nodes > STT_TREE_MAX_NODES)
    return stt_fail(STT_ERR_UNSUPPORTED, "%d nodes per tree: 1 to %d", a->max_nodes, STT_TREE_MAX_NODES);
  if ((int64_t)a->width * a->block_size > 0x7fffffff)
    return stt_fail(STT_ERR_UNSUPPORTED, "%d blocks of %d positions per sequence pass 2^31", a->width, a->block_size);
  return STT_OK;
}

// Query rows of a (sequence, KV head) at most, and the kernel variant that takes them.
struct TreeVariant { int nr, wr; };
TreeVariant tree_variant(const stt_tree_attention_args& a) {
  const int rows = a.max_nodes * (a.n_heads / a.n_kv_heads);
  if (rows <= 16) return {1, 1};
  if (rows <= 64) return {1, 4};
  if (rows <= 128) return {2, 4};
  return {4, 4};
}

TreeShape tree_shape(const stt_tree_attention_args& a) {
  TreeShape sh{};
  const TreeVariant v = tree_variant(a);
  const int rows = a.max_nodes * (a.n_heads / a.n_kv_heads), per = 16 * v.nr * v.wr;
  sh.row_tiles = (rows + per - 1) / per;
  int64_t keys = (int64_t)a.width * a.block_size;
  if (a.max_cached > 0 && a.max_cached < keys) keys = a.max_cached;
  const int64_t units = (int64_t)a.n_seq * a.n_kv_heads * sh.row_tiles;
  const int64_t target = 1024;
  int64_t chunk = (keys * units + target - 1) / target;
  chunk = (chunk + 127) / 128 * 128;
  if (chunk < 256) chunk = 256;
  sh.slices = keys > chunk ? (int)((keys + chunk - 1) / chunk) : 1;
  sh.chunk = (int)(chunk > 0x7fffff00 ? 0x7fffff00 : chunk);
  return sh;
}

template <typename T, int D>
void launch_tree(const stt_tree_attention_args& a, const TreeShape& sh, unsigned blocks, unsigned joins, hipStream_t st) {
  const TreeVariant v = tree_variant(a);
  // WIDE addresses a tile as one uniform base plus 32-bit lane offsets
  const bool wide = a.block_size >= kTile && a.pos_stride >= 0 && a.pos_stride < (1 << 25);
#define STT_TREE(NR, WR)                                                                                              \
  do {                                                                                                                \
    if (wide) hipLaunchKernelGGL((tree_attention_kernel<T, D, NR, WR, true>), dim3(blocks), dim3(256), 0, st, a, sh);  \
    else hipLaunchKernelGGL((tree_attention_kernel<T, D, NR, WR, false>), dim3(blocks), dim3(256), 0, st, a, sh);      \
  } while (0)
  if (v.wr == 1) STT_TREE(1, 1);
  else if (v.nr == 1) STT_TREE(1, 4);
  else if (v.nr == 2) STT_TREE(2, 4);
  else STT_TREE(4, 4);
#undef STT_TREE
  if (joins) hipLaunchKernelGGL((tree_join_kernel<T, D>), dim3(joins), dim3(D), 0, st, a, sh);
}

}  // namespace

extern "C" {

int stt_paged_plan(const int32_t* d_cached, const int32_t* d_new, int n_req, int block_size, int32_t* d_table,
                   int width, int32_t* d_free, int n_ring, const int64_t* d_ring_in, int64_t* d_ring_out,
                   const int32_t* d_held_in, int32_t* d_held_out, int rows, int32_t* d_starts, int64_t* d_slots,
                   int32_t* d_positions, int32_t* d_status, void* stream) {
  if (n_req < 1 || n_req > STT_PLAN_MAX_REQUESTS)
    return stt_fail(STT_ERR_UNSUPPORTED, "%d requests: 1 to %d", n_req, STT_PLAN_MAX_REQUESTS);
  if (!power_of_two(block_size) || block_size > 65536)
    return stt_fail(STT_ERR_UNSUPPORTED, "block size %d: a power of two <= 65536", block_size);
  if (width < 1 || n_ring < 1 || rows < 0 || (int64_t)width * block_size > 0x7fffffff)
    return stt_fail(STT_ERR_INVALID_ARGUMENT, "bad sizes (table width %d, ring %d, rows %d)", width, n_ring, rows);
  if (!d_cached || !d_new || !d_table || !d_free || !d_ring_in || !d_ring_out || !d_held_in || !d_held_out || !d_starts ||
      !d_status || (rows && (!d_slots || !d_positions)))
    return stt_fail(STT_ERR_INVALID_ARGUMENT, "null argument");
  if (d_ring_in == d_ring_out || d_held_in == d_held_out)
    return stt_fail(STT_ERR_INVALID_ARGUMENT, "the state before and after the step must be different buffers");
  PlanArgs a{d_cached, d_new, n_req, __builtin_ctz(block_size), d_table, width, d_free, n_ring, d_ring_in, d_ring_out,
             d_held_in, d_held_out, rows, d_starts, d_slots, d_positions, d_status, 1};
  const int avg = rows / n_req;
  while (a.group < 64 && a.group < avg) a.group <<= 1;
  const int64_t lanes = (int64_t)n_req * a.group;
  int64_t blocks = (lanes + kPlanThreads - 1) / kPlanThreads;
  blocks = blocks < 1 ? 1 : blocks > 256 ? 256 : blocks;
  hipLaunchKernelGGL(paged_plan_kernel, dim3((unsigned)blocks), dim3(kPlanThreads), 0, (hipStream_t)stream, a);
  STT_HIP_OR_FAIL(hipGetLastError(), (void)0);
  return STT_OK;
}

size_t stt_tree_attention_workspace_bytes(const stt_tree_attention_args* args) {
  if (check_tree(args) || args->n_seq == 0 || args->rows == 0) return 0;
  const TreeShape sh = tree_shape(*args);
  return sh.slices == 1 ? 0 : (size_t)args->rows * args->n_heads * sh.slices * (args->head_dim + 2) * sizeof(float);
}

int stt_tree_attention(const stt_tree_attention_args* a, void* d_workspace, size_t workspace_bytes, void* stream_) {
  hipStream_t st = (hipStream_t)stream_;
  const int rc = check_tree(a);
  if (rc) return rc;
  if (a->n_seq == 0 || a->rows == 0) return STT_OK;
  if (!a->d_q || !a->d_k || !a->d_v || !a->d_cached || !a->d_starts || !a->d_slots || !a->d_out ||
      (a->width && !a->d_table) || (a->n_blocks && (!a->d_k_cache || !a->d_v_cache)))
    return stt_fail(STT_ERR_INVALID_ARGUMENT, "null argument");
  const uintptr_t ptrs = (uintptr_t)a->d_q | (uintptr_t)a->d_k | (uintptr_t)a->d_v | (uintptr_t)a->d_k_cache |
                         (uintptr_t)a->d_v_cache | (uintptr_t)a->d_out;
  const int64_t strides = a->q_row | a->q_head | a->k_row | a->k_head | a->v_row | a->v_head | a->block_stride |
                          a->head_stride | a->pos_stride | a->out_row | a->out_head;
  if ((ptrs & 15) || (strides & 7))
    return stt_fail(STT_ERR_INVALID_ARGUMENT, "pointers must be 16-byte aligned and strides multiples of 8 elements");
  TreeShape sh = tree_shape(*a);
  const int64_t blocks = (int64_t)a->n_seq * a->n_kv_heads * sh.row_tiles * sh.slices;
  const int64_t joins = sh.slices == 1 ? 0 : (int64_t)a->n_seq * a->max_nodes * a->n_heads;
  if (blocks > 0x7fffffff || joins > 0x7fffffff)
    return stt_fail(STT_ERR_UNSUPPORTED, "%d sequences of %d heads exceed one launch", a->n_seq, a->n_heads);
  if (sh.slices > 1) {
    const size_t need = stt_tree_attention_workspace_bytes(a);
    if (!d_workspace || workspace_bytes < need || ((uintptr_t)d_workspace & 15))
      return stt_fail(STT_ERR_WORKSPACE, "workspace of %zu bytes, 16-byte aligned, needed (%zu given)", need, workspace_bytes);
    sh.part = (float*)d_workspace;
    sh.stat = sh.part + (size_t)a->rows * a->n_heads * sh.slices * a->head_dim;
  }
  if (a->dtype == STT_BF16) {
    if (a->head_dim == 64) launch_tree<__bf16, 64>(*a, sh, (unsigned)blocks, (unsigned)joins, st);
    else launch_tree<__bf16, 128>(*a, sh, (unsigned)blocks, (unsigned)joins, st);
  } else {
    if (a->head_dim == 64) launch_tree<_Float16, 64>(*a, sh, (unsigned)blocks, (unsigned)joins, st);
    else launch_tree<_Float16, 128>(*a, sh, (unsigned)blocks, (unsigned)joins, st);
  }
  STT_HIP_OR_FAIL(hipGetLastError(), (void)0);
  return STT_OK;
}

}  // extern "C"
