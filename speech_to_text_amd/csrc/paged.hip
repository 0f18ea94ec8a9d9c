// Paged K/V cache: block tables and slot maps from request lengths, and attention of drafted token
// trees over the cache (stt_paged_plan, stt_tree_attention of include/stt_mi355x.h).
#include <algorithm>
#include "paged.h"
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
//   Bound by dependent memory round trips, not by bytes (lengths, lengths again where a request is served, table
// and ring entries): 8 requests 5.9 us, 2 048 requests with half a million new rows (6.8 MB, 1.3 us at the copy
// rate) 11.8 us.
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
// Keys come in tiles of 32: the tree's own nodes (last slice), whose K/V the block also stores into the
// cache, then cached positions.  Per tile, S^T = K Q^T and O^T += V^T P^T on the matrix cores
// (v_mfma_f32_16x16x32): a lane holds one query against 8 keys, so maximum, sum and rescale factor
// are per lane; the two score products of a tile take the keys 8a + b and 8a + 4 + b (a, b < 4), so
// that the exponentiated scores of lane group g are the keys 8g .. 8g + 7 in order and, in the
// storage type (what the matrix cores take), already are the B operand of the second product.  That is done
// twice: a weight is the sum of its rounding to the storage type and of the remainder's (bf16 2^-16 of the weight at
// most is lost, fp16 2^-22), since one rounding alone would cost as much as the result's own.  K and V go through LDS
// images as they come from memory; V is read back transposed.
//   The softmax keeps a reference r <= max <= r + 8 per query (base-2 units): it is moved, and the sums
// rescaled, only when a tile raises the maximum more than 8 above it, so weights are at most 2^8.  fp16 weights
// carry 2^7 more, which the normaliser has as well: the type ends at 2^16, and its smallest step of 2^-24 then is 2^-31
// of the largest key's weight.
//   A value that is not finite makes these products infinite or NaN where a query sees it or not, whatever
// its weight.  Sums that end so are made again from the start with every tile taken as one of nodes (SPOILED below).
//   WR = 1: each of WV waves walks its own tiles (every WV-th) for all 16 NR rows of the block, staging
// through wave-private images without barriers, and the waves' (reference, sum, O) are joined at the end: few rows,
// memory bound, so that the second product of the weights costs nothing.  600 ragged windows x 20 heads x 9-16 nodes
// (779 MB) 159 us, 4.9 TB/s; 48 requests of up to 16 000 positions, one node (1.6 GB) 271 us, 5.9 TB/s.
//   WR = 4, 8: the waves share each tile and own 16 NR rows each, so that K and V are read once for 64, 128 or
// 256 rows.  131 000 positions x 64 nodes x 32 heads of 128 240 us, 572 TFLOP/s (with weights of one rounding a call
// took 196 us, now 246): bound by the instructions of two waves a SIMD (matrix 38 %, vector 47 % of the cycles),
// which overlap little; registers leave no third wave.
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
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(pa_f2{a, b}, pa_b2)); }
  static __device__ __forceinline__ pa_f4 mfma(pa_u4 a, pa_u4 b, pa_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_b8, a), __builtin_bit_cast(pa_b8, b), c, 0, 0, 0);
  }
  // what the two halves of a packed pair stand for
  static __device__ __forceinline__ float low(uint32_t u) { return __uint_as_float(u << 16); }
  static __device__ __forceinline__ float high(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }
  static constexpr uint32_t kExponent = 0x7F80, kOne = 0x3F80, kMinusMark = 0x4300, kNanMark = 0x4680;   // 1, 128, 16384
  static constexpr float kLift = 0.f;                // weights are multiplied by 2^kLift
};
template <> struct Half<_Float16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(pa_f2{a, b}, pa_h2)); }
  static __device__ __forceinline__ pa_f4 mfma(pa_u4 a, pa_u4 b, pa_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pa_h8, a), __builtin_bit_cast(pa_h8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float low(uint32_t u) { return (float)__builtin_bit_cast(pa_h2, u)[0]; }
  static __device__ __forceinline__ float high(uint32_t u) { return (float)__builtin_bit_cast(pa_h2, u)[1]; }
  static constexpr uint32_t kExponent = 0x7C00, kOne = 0x3C00, kMinusMark = 0x5800, kNanMark = 0x7400;
  static constexpr float kLift = 7.f;
};

// f v; infinities and NaN stay what they are where f has underflowed to zero
__device__ __forceinline__ pa_f4 scaled(pa_f4 v, float f) {
  pa_f4 y;
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = f == 0.f ? (fabsf(v[r]) < __builtin_inff() ? 0.f : v[r]) : f * v[r];
  return y;
}

struct TreeShape {
  int chunk;        // cached positions per slice, a multiple of 32
  int slices;       // slices in the grid; a sequence uses ceil(cached / chunk) of them, at least one
  int row_tiles;    // blocks per (sequence, KV head, slice)
  uint32_t units;   // n_seq x KV heads x slices
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
constexpr int kManyUnits = 2048;

// One wave's queries and running sums, and the work on one 32-key tile.
// SPREAD: images without bank conflicts, for the variants whose waves share them.
template <typename T, int D, int NR, bool SPREAD>
struct TreeWave {
  // Key rows of the images.  64 banks of 4 bytes: 16 lanes of a K read (rows 8 a + b, a and b below 4, 16
  // bytes each) and 32 lanes of a transposed V read (rows 8 a + b, a below 2, 32 bytes each) meet every bank once
  // with the SPREAD pitches and a shift every 16 rows of K and every 8 rows of V.  With plain rows each of
  // these reads takes twice as long.  A wave that streams its own tiles waits for memory, not for them, and
  // has no registers for a second set of addresses.
  static constexpr int kPitchK = 2 * D + 16, kShiftK = SPREAD ? 64 : 0;
  static constexpr int kPitchV = 2 * D + (SPREAD ? 32 : 16), kShiftV = SPREAD ? 128 : 0;
  static constexpr int kImage = kTile * kPitchV + 3 * kShiftV;
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

  // Two stored values without their infinities and NaNs; `count` receives what those count as.  Halves
  // are compared by carries: magnitude + (0x8000 - exponent mask) reaches bit 15 where the exponent is
  // all ones, one less where the mantissa is not zero either; (bit 0 | bit 16) * 0xFFFF spreads the answer.
  static __device__ __forceinline__ uint32_t split(uint32_t u, uint32_t& count) {
    constexpr uint32_t both = 0x00010001u, e = Half<T>::kExponent;
    const uint32_t mag = u & (0x7FFFu * both);
    const uint32_t odd = (((mag + (0x8000u - e) * both) >> 15) & both) * 0xFFFFu;
    const uint32_t nan = (((mag + (0x7FFFu - e) * both) >> 15) & both) * 0xFFFFu;
    const uint32_t minus = ((u >> 15) & both) * 0xFFFFu;
    count = (nan & (Half<T>::kNanMark * both)) | (odd & ~nan & ((minus & (Half<T>::kMinusMark * both)) | (~minus & (Half<T>::kOne * both))));
    return u & ~odd;
  }
  // 1.0 for each of the two lowest bits that is set
  static __device__ __forceinline__ uint32_t ones(uint32_t bits) {
    return (bits & 1u) * Half<T>::kOne | ((bits >> 1) & 1u) * (Half<T>::kOne << 16);
  }

  // Whether some sum is infinite or NaN (0 * that is not 0)
  __device__ __forceinline__ bool spoiled() const {
    float odd = 0.f;
#pragma unroll
    for (int x = 0; x < NR; ++x)
#pragma unroll
      for (int t = 0; t < D / 16; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) odd = __builtin_fmaf(o[x][t][r], 0.f, odd);
    return !(odd == 0.f);
  }

  // History tiles: bit l of `ok` says whether key l exists; the K and V of the others are zero.  TREE: bit j
  // of keep[x] says whether the lane's query x sees key 8 g + j; K and V of keys it does not see may be anything.
  // SPOILED: some value of the tile is not finite and may belong to a key a query does not see; a zero
  // weight would still turn it into NaN on the matrix cores.  Then the finite values are multiplied
  // alone, a second product counts the infinities and NaNs among the keys a query does see (exact
  // small integers: +inf 1, -inf 128, NaN 16384, at most 32 keys), and those are added afterwards.
  template <bool TREE, bool SPOILED>
  __device__ __forceinline__ void tile(const unsigned char* kimg, const unsigned char* vimg, uint32_t ok,
                                       const uint32_t (&keep)[NR], float scale2, int lane) {
    const int col = lane & 15, g = lane >> 4;
    const unsigned char* ka = kimg + (8 * (col >> 2) + (col & 3)) * kPitchK + (col >> 3) * kShiftK + 16 * g;
    pa_f4 s1[NR], s2[NR];
#pragma unroll
    for (int x = 0; x < NR; ++x) s1[x] = s2[x] = pa_f4{0.f, 0.f, 0.f, 0.f};
    if (SPREAD && !TREE) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const pa_u4 a0 = *(const pa_u4*)(ka + 64 * c), a1 = *(const pa_u4*)(ka + 4 * kPitchK + 64 * c);
#pragma unroll
      for (int x = 0; x < NR; ++x) {
        s1[x] = Half<T>::mfma(a0, q[x][c], s1[x]);
        s2[x] = Half<T>::mfma(a1, q[x][c], s2[x]);
      }
      if (TREE) __builtin_amdgcn_sched_barrier(0);   // (few registers rather than early reads: one or two tiles a block)
    }
    if (TREE && NR * D > 128) __builtin_amdgcn_sched_barrier(0);
    // transposed read: lane 4 u + w of a 16-lane group addresses key row 8 g + 4 half + u, features
    // 16 t + 4 w ..; lane i receives feature 16 t + i of the four keys
    auto values = [&](int t) __attribute__((always_inline)) {
      const unsigned char* at = vimg + (8 * g + (col >> 2)) * kPitchV + g * kShiftV + (16 * t + 4 * (col & 3)) * 2;
      const pa_u2 lo = __builtin_bit_cast(pa_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)at));
      const pa_u2 hi = __builtin_bit_cast(pa_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s4*)(at + 4 * kPitchV)));
      return pa_u4{lo.x, lo.y, hi.x, hi.y};
    };
    if (SPREAD && !TREE) __builtin_amdgcn_s_setprio(0);
    constexpr int kEarly = TREE || !SPREAD ? 0 : NR * D > 128 ? D / 32 : D / 16;
    pa_u4 early[kEarly ? kEarly : 1];
#pragma unroll
    for (int t = 0; t < kEarly; ++t) early[t] = values(t);
    pa_u4 pf[NR], pl[NR];                              // weights: rounded, and what that left
#pragma unroll
    for (int x = 0; x < NR; ++x) {
      float z[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) { z[r] = s1[x][r]; z[4 + r] = s2[x][r]; }
      if (TREE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = (keep[x] >> j) & 1 ? z[j] : -__builtin_inff();
      } else if (ok != 0xFFFFFFFFu) {
        const uint32_t mine = ok >> (8 * g);
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = (mine >> j) & 1 ? z[j] : -__builtin_inff();
      }
      float top = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7]))) * scale2;
      if (__any(top > ref[x] + 8.0f)) {              // only then do the lanes of a query talk to each other
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (top > ref[x] + 8.0f) {                   // (from -inf: nothing seen yet, the sums are zero)
          const float f = __builtin_amdgcn_exp2f(ref[x] - top);
          ref[x] = top;
          sum[x] *= f;
#pragma unroll
          for (int t = 0; t < D / 16; ++t) o[x][t] = SPOILED ? scaled(o[x][t], f) : o[x][t] * f;
        }
      }
      const float base = Half<T>::kLift - (ref[x] == -__builtin_inff() ? 0.f : ref[x]);
#pragma unroll
      for (int j = 0; j < 8; ++j) z[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[j], scale2, base));
      sum[x] += ((z[0] + z[1]) + (z[2] + z[3])) + ((z[4] + z[5]) + (z[6] + z[7]));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t near = Half<T>::pack(z[2 * j], z[2 * j + 1]);
        pf[x][j] = near;
        pl[x][j] = Half<T>::pack(z[2 * j] - Half<T>::low(near), z[2 * j + 1] - Half<T>::high(near));
      }
    }
    // (a tree tile of the largest variant cannot hold the next phase's operands as well)
    if (TREE && NR * D > 128) __builtin_amdgcn_sched_barrier(0);
    if (SPREAD && !TREE) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      pa_u4 v = t < kEarly ? early[t < kEarly ? t : 0] : values(t);
      if (SPOILED) {
        uint32_t c0, c1, c2, c3;
        v = pa_u4{split(v.x, c0), split(v.y, c1), split(v.z, c2), split(v.w, c3)};
        const pa_u4 count = {c0, c1, c2, c3};
#pragma unroll
        for (int x = 0; x < NR; ++x) {
          const pa_u4 sees = {ones(keep[x]), ones(keep[x] >> 2), ones(keep[x] >> 4), ones(keep[x] >> 6)};
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
#pragma unroll
      for (int x = 0; x < NR; ++x) o[x][t] = Half<T>::mfma(v, pl[x], o[x][t]);
      if (TREE) __builtin_amdgcn_sched_barrier(0);
    }
    if (SPREAD && !TREE) __builtin_amdgcn_s_setprio(0);
  }
};

// 16-byte pieces of one key tile as a group of LANES threads holds them: piece = key * (D / 8) + part.
// APART: one half of the threads holds K, the other half V (LANES counts one half).
template <int D, int LANES, bool APART>
struct TilePieces {
  static constexpr int kPer = kTile * (D / 8) / LANES;
  static constexpr int kKeysPerStep = LANES / (D / 8);
  pa_u4 k[kPer], v[APART ? 1 : kPer];                // (APART: k is whichever of the two)
};

template <typename T, int D, int NR, int WR, int WV, bool PAGED>
__global__ __launch_bounds__(64 * WV, NR == 1 && D == 64 ? 3 : 2) void tree_attention_kernel(
    const stt_tree_attention_args a, const TreeShape sh) {
  typedef TreeWave<T, D, NR, (WR > 1)> Wave;
  constexpr int LANES = WR == 1 ? 64 : 256;          // threads that load a tile together
  constexpr bool STREAM = WR == 1;                   // nobody else reads these positions
  constexpr bool APART = WR == 8;
  typedef TilePieces<D, LANES, APART> Pieces;
  __shared__ __attribute__((aligned(16))) unsigned char lds[WR == 1 ? 2 * WV : 4][Wave::kImage];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g = lane >> 4;
  // Blocks go to the eight XCDs round robin: the row tiles of one slice, which read the same K/V, are
  // numbered eight apart so that they share an L2.
  uint32_t id = blockIdx.x;
  int rt = 0;
  if (sh.row_tiles > 1) {
    const uint32_t eight = id / (8 * sh.row_tiles), in = id - eight * (8 * sh.row_tiles);
    rt = (int)(in >> 3);
    id = eight * 8 + (in & 7);
    if (id >= sh.units) return;
  }
  const int slice = (int)(id % (uint32_t)sh.slices);
  id /= (uint32_t)sh.slices;
  const int hk = (int)(id % (uint32_t)a.n_kv_heads), seq = (int)(id / (uint32_t)a.n_kv_heads);
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
  const int tiles = (key1 - key0 + kTile - 1) / kTile;
  const int tree_tiles = slice == used - 1 ? (nodes + kTile - 1) / kTile : 0;
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
    if (a.scale < 0.f) {                             // the sign goes to the queries: maxima stay maxima
#pragma unroll
      for (int c = 0; c < D / 32; ++c) w.q[x][c] ^= 0x80008000u;
    }
  }
  // (a scale of zero becomes a tiny one: scores stay at zero and -inf stays -inf)
  const float scale2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-37f);

  const half_bits* kc = (const half_bits*)a.d_k_cache + hk * a.head_stride;
  const half_bits* vc = (const half_bits*)a.d_v_cache + hk * a.head_stride;
  const int loader = WR == 1 ? lane : tid & (LANES - 1), load_wave = WR == 1 ? 0 : wave & (LANES / 64 - 1);
  const bool load_v = APART && wave >= LANES / 64;    // (a whole wave's)
  const half_bits* mine_c = load_v ? vc : kc;
  const int piece = loader % (D / 8), key_in = loader / (D / 8);

  // Block ids: lane l < 32 holds the one of the tile's position l, -1 where the table has none.
  const int32_t* table = a.d_table + (long)seq * a.width;
  // Tiles past the end are fetched as the last one again: with a branch around a load the compiler has to
  // assume the worst about what is in flight and waits for all of it.
  auto within = [&](int t) __attribute__((always_inline)) { return t < tiles ? t : tiles - 1; };
  auto load_ids = [&](int t) __attribute__((always_inline)) -> int {
    const int at = (key0 + t * kTile + (lane & 31)) >> shift;
    const int id = table[at < a.width ? at : a.width - 1];
    return at < a.width ? id : -1;
  };
  // PAGED: one load instruction of a wave covers 512 / D positions, all in one block, so that the block's
  // base is a scalar and the lanes add a constant 32-bit offset.
  const uint32_t lane_off = (uint32_t)((lane / (D / 8)) * (int)a.pos_stride + 8 * piece);
  auto load = [&](int t, int ids, Pieces& p) __attribute__((always_inline)) {
    const int pos = key0 + t * kTile;
    const int use = (uint32_t)ids < (uint32_t)a.n_blocks ? ids : 0;
#pragma unroll
    for (int i = 0; i < Pieces::kPer; ++i) {
      const pa_u4 *kp, *vp;
      if (PAGED) {
        const int key = load_wave * (512 / D) + i * Pieces::kKeysPerStep;
        const long at = (long)__builtin_amdgcn_readlane(use, key) * a.block_stride + (long)((pos + key) & (a.block_size - 1)) * a.pos_stride;
        kp = (const pa_u4*)((APART ? mine_c : kc) + at + lane_off);
        vp = (const pa_u4*)(vc + at + lane_off);
      } else {
        const int key = key_in + i * Pieces::kKeysPerStep;
        const long at = __shfl(use, key, 64) * a.block_stride + (long)((pos + key) & (a.block_size - 1)) * a.pos_stride + 8 * piece;
        kp = (const pa_u4*)((APART ? mine_c : kc) + at);
        vp = (const pa_u4*)(vc + at);
      }
      if (STREAM) { p.k[i] = __builtin_nontemporal_load(kp); p.v[APART ? 0 : i] = __builtin_nontemporal_load(vp); }
      else { p.k[i] = *kp; if (!APART) p.v[APART ? 0 : i] = *vp; }
    }
  };
  // registers -> LDS images
  auto put = [&](const Pieces& p, unsigned char* kimg, unsigned char* vimg) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < Pieces::kPer; ++i) {
      // (key_in is below kKeysPerStep, a power of two: the shifts of the sum are the sums of the shifts)
      const int more = i * Pieces::kKeysPerStep, key = key_in + more;
      const int in_k = key * Wave::kPitchK + ((key_in >> 4) + (more >> 4)) * Wave::kShiftK + 16 * piece;
      const int in_v = key * Wave::kPitchV + ((key_in >> 3) + (more >> 3)) * Wave::kShiftV + 16 * piece;
      if (APART) {
        *(pa_u4*)(load_v ? vimg + in_v : kimg + in_k) = p.k[i];
      } else {
        *(pa_u4*)(kimg + in_k) = p.k[i];
        *(pa_u4*)(vimg + in_v) = p.v[APART ? 0 : i];
      }
    }
  };
  // Tile t of the cached positions: which of them exist (not those behind the history or without a block);
  // the others get zero K and V.
  auto present = [&](int t, int ids) __attribute__((always_inline)) {
    return (uint32_t)__ballot(key0 + t * kTile + (lane & 31) < key1 && (uint32_t)ids < (uint32_t)a.n_blocks);
  };
  auto stage = [&](uint32_t ok, Pieces& p, unsigned char* kimg, unsigned char* vimg) __attribute__((always_inline)) {
    if (ok != 0xFFFFFFFFu) {
#pragma unroll
      for (int i = 0; i < Pieces::kPer; ++i)
        if (!((ok >> (key_in + i * Pieces::kKeysPerStep)) & 1)) p.k[i] = p.v[APART ? 0 : i] = pa_u4{0, 0, 0, 0};
    }
    put(p, kimg, vimg);
  };
  // The tree's own nodes u * 32 ..: into the cache (one row tile does it) and into the images.  True for
  // threads that met a value that is not finite.
  auto stage_nodes = [&](int u, unsigned char* kimg, unsigned char* vimg) __attribute__((always_inline)) -> bool {
    Pieces p;
    bool odd = false;
    // (opaque, so that addresses are worked out here and do not take registers all through the loop around)
    int key_here = key_in, piece_here = piece;
    asm volatile("" : "+v"(key_here), "+v"(piece_here));
#pragma unroll
    for (int i = 0; i < Pieces::kPer; ++i) {
      const int want = u * kTile + key_here + i * Pieces::kKeysPerStep, nd = want < nodes ? want : nodes - 1;
      const half_bits* kn = (const half_bits*)a.d_k + (long)(row0 + nd) * a.k_row + hk * a.k_head + 8 * piece_here;
      const half_bits* vn = (const half_bits*)a.d_v + (long)(row0 + nd) * a.v_row + hk * a.v_head + 8 * piece_here;
      p.k[i] = *(const pa_u4*)(load_v ? vn : kn);
      if (!APART) p.v[APART ? 0 : i] = *(const pa_u4*)vn;
    }
#pragma unroll
    for (int i = 0; i < Pieces::kPer; ++i) {
      const int want = u * kTile + key_here + i * Pieces::kKeysPerStep;
      constexpr uint32_t e = Half<T>::kExponent;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t vw = APART ? p.k[i][j] : p.v[APART ? 0 : i][j];      // (K that is not finite only costs time)
        odd |= (vw & e) == e || (vw & (e << 16)) == (e << 16);
      }
      if (rt == 0 && want < nodes) {
        const long slot = a.d_slots[row0 + want];
        if (slot >= 0 && slot < ((long)a.n_blocks << shift)) {
          const long at = (slot >> shift) * a.block_stride + hk * a.head_stride + (slot & (a.block_size - 1)) * a.pos_stride + 8 * piece_here;
          *(pa_u4*)((half_bits*)(load_v ? a.d_v_cache : a.d_k_cache) + at) = p.k[i];
          if (!APART) *(pa_u4*)((half_bits*)a.d_v_cache + at) = p.v[APART ? 0 : i];
        }
      }
    }
    put(p, kimg, vimg);
    return odd;
  };
  auto seen_nodes = [&](int u, unsigned long long path, uint32_t (&keep)[NR]) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < NR; ++x) keep[x] = (uint32_t)(__shfl(path, node[x], 64) >> (u * kTile + 8 * g)) & 255u;
  };
  auto tree_tile = [&](int u, unsigned long long path, bool spoiled, const unsigned char* kimg, const unsigned char* vimg) __attribute__((always_inline)) {
    uint32_t keep[NR];
    seen_nodes(u, path, keep);
    if (spoiled) w.template tile<true, true>(kimg, vimg, 0u, keep, scale2, lane);
    else w.template tile<true, false>(kimg, vimg, 0u, keep, scale2, lane);
  };

  const uint32_t all[NR] = {};                       // (history tiles do not look at it)
  // The tree's tiles go first (WR = 1: while the first loads of the history are on their way).
  if (WR == 1) {
    // Two register sets alternate between "in flight" and "being used"; block ids are fetched one
    // tile further ahead, since the addresses of the next loads wait for them.
    unsigned char *kimg = lds[2 * wave], *vimg = lds[2 * wave + 1];
    Pieces pa, pb;
    uint32_t ok;
    int ia = -1, ib = -1;
    if (wave < tiles) {
      ia = load_ids(wave);
      ib = load_ids(within(wave + WV));
      load(wave, ia, pa);
    }
    if (wave < tree_tiles) {
      const unsigned long long path = tree_path(a.d_parents, row0, nodes, lane);
#pragma unroll 1
      for (int u = wave; u < tree_tiles; u += WV) {
        const bool odd = __any(stage_nodes(u, kimg, vimg));
        tree_tile(u, path, odd, kimg, vimg);
      }
    }
    int t = wave;
    for (; t + WV < tiles; t += 2 * WV) {
      const int ia2 = load_ids(within(t + 2 * WV)), ib2 = load_ids(within(t + 3 * WV));
      load(t + WV, ib, pb);
      stage(ok = present(t, ia), pa, kimg, vimg);
      w.template tile<false, false>(kimg, vimg, ok, all, scale2, lane);
      load(within(t + 2 * WV), ia2, pa);
      stage(ok = present(t + WV, ib), pb, kimg, vimg);
      w.template tile<false, false>(kimg, vimg, ok, all, scale2, lane);
      ia = ia2; ib = ib2;
    }
    if (t < tiles) {
      stage(ok = present(t, ia), pa, kimg, vimg);
      w.template tile<false, false>(kimg, vimg, ok, all, scale2, lane);
    }
  } else {
    // Tile t goes through images (t & 1); the kAhead tiles behind the next are on their way to registers.
    constexpr int kAhead = APART ? 2 : NR * D > 128 ? 1 : 2;
    if (tree_tiles) {
      const unsigned long long path = tree_path(a.d_parents, row0, nodes, lane);
#pragma unroll 1
      for (int u = 0; u < tree_tiles; ++u) {
        const bool odd = __syncthreads_or(stage_nodes(u, lds[2 * u], lds[2 * u + 1]));
        tree_tile(u, path, odd, lds[2 * u], lds[2 * u + 1]);
      }
      __syncthreads();
    }
    if (tiles > 0) {
      Pieces p[kAhead];
      uint32_t ok[kAhead];                             // bit l: position l of the tile exists
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int id = load_ids(within(u));
        ok[u] = present(u, id);
        load(within(u), id, p[u]);
      }
      // Block ids run kAhead tiles before the loads that need them: loads return in order, so that a wait
      // for one that was issued last would be a wait for all (32 sequences of up to 4 000 keys x 64 nodes: 217 us, so 202).
      int ids[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) ids[u] = load_ids(within(kAhead + u));
      auto refill = [&](int t, int u) __attribute__((always_inline)) {     // p[u] with tile t
        const int use = ids[u];
        ids[u] = load_ids(within(t + kAhead));
        ok[u] = present(t, use);
        load(within(t), use, p[u]);
      };
      uint32_t now = ok[0];
      stage(now, p[0], lds[0], lds[1]);
      refill(kAhead, 0);
      lds_barrier();
      // Tile t from its images while tile t + 1 goes to the others, which were last read before the barrier
      // of tile t - 1; one barrier a tile, and its wait for the writes is over by then.
      auto step = [&](int t, int phase) __attribute__((always_inline)) {
        const int u = (phase + 1) % kAhead, image = phase & 1;
        const uint32_t then = ok[u];
        stage(then, p[u], lds[2 - 2 * image], lds[3 - 2 * image]);
        refill(t + 1 + kAhead, u);
        w.template tile<false, false>(lds[2 * image], lds[2 * image + 1], now, all, scale2, lane);
        now = then;
        lds_barrier();
      };
      int t = 0;
      for (; t + 2 <= tiles; t += 2) {
        step(t, 0);
        step(t + 1, 1);
      }
      if (t < tiles) step(t, 0);
    }
  }

  // Sums that are not finite: the same tiles again (a wave's own, where it walks alone), their values split.  Rare, so one at
  // a time.
  auto again = [&](int first, int step, unsigned char* kimg, unsigned char* vimg) __attribute__((always_inline)) {
    const unsigned long long path = tree_tiles ? tree_path(a.d_parents, row0, nodes, lane) : 0ull;
    w.clear();
    bool history = false;
#pragma unroll 1
    for (int u = first;; u += step) {
      if (!history && u >= tree_tiles) { history = true; u = first; }
      if (history && u >= tiles) break;
      if (WR > 1) __syncthreads();                     // the images are read
      uint32_t keep[NR];
      if (!history) {
        stage_nodes(u, kimg, vimg);
        seen_nodes(u, path, keep);
      } else {
        Pieces p;
        const int ids = load_ids(u);
        const uint32_t ok = present(u, ids);
        load(u, ids, p);
        stage(ok, p, kimg, vimg);
#pragma unroll
        for (int x = 0; x < NR; ++x) keep[x] = (ok >> (8 * g)) & 255u;
      }
      if (WR > 1) __syncthreads();
      w.template tile<true, true>(kimg, vimg, 0u, keep, scale2, lane);
    }
  };
  if (WR == 1) {
    if (__any(w.spoiled())) again(wave, WV, lds[2 * wave], lds[2 * wave + 1]);
  } else {
    if (__syncthreads_or(w.spoiled())) again(0, 1, lds[0], lds[1]);
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
    if (WR > 1 || WV == 1) {
      const int r = wave_row + 16 * x + col;
      if (r < n_rows) {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) write(r, w.ref[x], sum, 16 * t + 4 * g, w.o[x][t]);
      }
      continue;
    }
    // join the waves: [query][feature] of each in its own images, then (reference, sum)
    float* mine = (float*)lds[2 * wave];
    constexpr int kRow = D + 4;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < D / 16; ++t) *(pa_f4*)(mine + col * kRow + 16 * t + 4 * g) = w.o[x][t];
    if (g == 0) { mine[16 * kRow + col] = w.ref[x]; mine[16 * kRow + 16 + col] = sum; }
    __syncthreads();
    for (int e = tid; e < 16 * (D / 4); e += 64 * WV) {
      const int qi = e / (D / 4), f = 4 * (e % (D / 4));
      const int r = first_row + 16 * x + qi;
      if (r >= n_rows) continue;
      float rf[WV], top = -__builtin_inff();
#pragma unroll
      for (int u = 0; u < WV; ++u) { rf[u] = ((const float*)lds[2 * u])[16 * kRow + qi]; top = fmaxf(top, rf[u]); }
      pa_f4 num = {0.f, 0.f, 0.f, 0.f};
      float den = 0.f;
#pragma unroll
      for (int u = 0; u < WV; ++u) {
        const float* src = (const float*)lds[2 * u];
        const float f2 = rf[u] == -__builtin_inff() ? (src[16 * kRow + 16 + qi] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(rf[u] - top);
        num += scaled(*(const pa_f4*)(src + qi * kRow + f), f2);
        if (f2 != 0.f) den += f2 * src[16 * kRow + 16 + qi];
      }
      write(r, top, den, f, num);
    }
  }
}

// Joins the slices of a (row, head) in slice order, so that results do not depend on the run.  Bound by one pass over
// the slices' sums (34 MB of 2 048 rows x 32 slices x 128: 10 us).  One wave each: lane = slice while the factors are
// worked out (64 at a time), then lane = 16-byte piece of the sums, 256 / D slices side by side.
template <typename T, int D>
__global__ __launch_bounds__(64) void tree_join_kernel(const stt_tree_attention_args a, const TreeShape sh) {
  constexpr int SIDE = 256 / D;                      // slices one wave load covers
  const int lane = threadIdx.x, f = 4 * (lane % (D / 4)), side = lane / (D / 4);
  uint32_t id = blockIdx.x;
  const int h = (int)(id % (uint32_t)a.n_heads);
  id /= (uint32_t)a.n_heads;
  const int node = (int)(id % (uint32_t)a.max_nodes), seq = (int)(id / (uint32_t)a.max_nodes);
  const int row0 = a.d_starts[seq];
  int nodes = a.d_starts[seq + 1] - row0;
  nodes = nodes < a.max_nodes ? nodes : a.max_nodes;
  if (node >= nodes || row0 < 0 || row0 > a.rows - nodes) return;
  const int used = tree_slices(tree_history(a, seq), sh);
  if (used == 1) return;
  const long at = ((long)(row0 + node) * a.n_heads + h) * sh.slices;
  float top = -__builtin_inff();
  for (int s = lane; s < used; s += 64) top = fmaxf(top, sh.stat[2 * (at + s)]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  pa_f4 num = {0.f, 0.f, 0.f, 0.f};
  float den = 0.f;
  for (int s0 = 0; s0 < used; s0 += 64) {
    float w = 0.f, l = 0.f;
    if (s0 + lane < used) {
      const float rf = sh.stat[2 * (at + s0 + lane)];
      l = sh.stat[2 * (at + s0 + lane) + 1];
      w = rf == -__builtin_inff() ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(rf - top);
    }
    const int n = used - s0 < 64 ? used - s0 : 64;
#pragma unroll 8
    for (int s = 0; s < n; s += SIDE) {
      const int mine = s + side < n ? s + side : n - 1;
      float ws = __shfl(w, mine, 64);
      if (s + side >= n) ws = 0.f;
      const pa_f4 v = *(const pa_f4*)(sh.part + (at + s0 + mine) * D + f);
      num += scaled(v, ws);                          // (a slice that saw nothing left its sums at zero)
    }
    den += w == 0.f ? 0.f : w * l;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) den += __shfl_xor(den, o, 64);
#pragma unroll
  for (int o = D / 4; o < 64; o <<= 1)
#pragma unroll
    for (int r = 0; r < 4; ++r) num[r] += __shfl_xor(num[r], o, 64);
  if (side == 0) {
    const float inv = 1.0f / den;
    half_bits* out = (half_bits*)a.d_out + (row0 + node) * a.out_row + h * a.out_head + f;
    *(pa_u2*)out = pa_u2{Half<T>::pack(num[0] * inv, num[1] * inv), Half<T>::pack(num[2] * inv, num[3] * inv)};
  }
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
struct TreeVariant { int nr, wr, wv; };
TreeVariant tree_variant(const stt_tree_attention_args& a) {
  const int rows = a.max_nodes * (a.n_heads / a.n_kv_heads);
  if (rows <= 16) return {1, 1, (int64_t)a.n_seq * a.n_kv_heads >= kManyUnits ? 1 : 4};
  if (rows <= 64) return {1, 4, 4};
  return rows <= 128 ? TreeVariant{2, 4, 4} : TreeVariant{2, 8, 8};
}

TreeShape tree_shape(const stt_tree_attention_args& a) {
  TreeShape sh{};
  const TreeVariant v = tree_variant(a);
  const int rows = a.max_nodes * (a.n_heads / a.n_kv_heads), per = 16 * v.nr * v.wr;
  sh.row_tiles = (rows + per - 1) / per;
  int64_t keys = (int64_t)a.width * a.block_size;
  if (a.max_cached > 0 && a.max_cached < keys) keys = a.max_cached;
  const int64_t pairs = (int64_t)a.n_seq * a.n_kv_heads;
  // Slices of equal length.  Row tiles that share images: the blocks that are resident together, one (eight
  // waves) or two on each of 256 compute units: a wave takes 1.2 us for a tile however many others there are,
  // and each slice more costs 8 D bytes per row, written and read.  One row tile: up to 2 048 blocks as long as
  // each has 2 048 keys, which evens out sequences of different lengths; down to 512 blocks otherwise.  No
  // slice is shorter than what its join costs.  Measured with D = 128 and 8 KV heads, us (another choice in
  // brackets): 131 000 keys, 256 rows 288 (512 blocks: 311), 64 rows 121 (2 048: 204), 16 rows 103 (2 048: 151);
  // 16 000 keys, 256 rows 60 (slices of 4 096: 206); 48 sequences of up to 16 000 keys 273 (512: 370).
  const int64_t total = keys * pairs * sh.row_tiles;
  auto over = [&](int64_t blocks) { return (total + blocks - 1) / blocks; };
  int64_t chunk = v.wr == 8 ? over(256) : v.wr == 4 ? over(512) : std::max<int64_t>(over(2048), std::min<int64_t>(over(512), 2048));
  chunk = std::max<int64_t>(chunk, v.wr == 1 ? 512 : 256);
  chunk = (chunk + 127) / 128 * 128;
  sh.slices = keys > chunk ? (int)((keys + chunk - 1) / chunk) : 1;
  sh.chunk = (int)(chunk > 0x7fffff00 ? 0x7fffff00 : chunk);
  const int64_t units = pairs * sh.slices;
  sh.units = (uint32_t)(units > 0xffffffff ? 0xffffffff : units);
  return sh;
}

template <typename T, int D>
void launch_tree(const stt_tree_attention_args& a, const TreeShape& sh, unsigned blocks, unsigned joins, hipStream_t st) {
  const TreeVariant v = tree_variant(a);
  // a wave load stays inside one block, and lane offsets inside 32 bits
  const bool paged = a.block_size >= 512 / D && a.pos_stride >= 0 && a.pos_stride < (1 << 25);
#define STT_TREE(NR, WR, WV)                                                                                          \
  do {                                                                                                                \
    if (paged) hipLaunchKernelGGL((tree_attention_kernel<T, D, NR, WR, WV, true>), dim3(blocks), dim3(64 * WV), 0, st, a, sh);  \
    else hipLaunchKernelGGL((tree_attention_kernel<T, D, NR, WR, WV, false>), dim3(blocks), dim3(64 * WV), 0, st, a, sh);      \
  } while (0)
  if (v.wr == 1) { if (v.wv == 1) STT_TREE(1, 1, 1); else STT_TREE(1, 1, 4); }
  else if (v.nr == 1) STT_TREE(1, 4, 4);
  else if (v.wr == 4) STT_TREE(2, 4, 4);
  else STT_TREE(2, 8, 8);
#undef STT_TREE
  if (joins) hipLaunchKernelGGL((tree_join_kernel<T, D>), dim3(joins), dim3(64), 0, st, a, sh);
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
  int64_t blocks = (int64_t)a->n_seq * a->n_kv_heads * sh.slices;
  if (sh.row_tiles > 1) blocks = (blocks + 7) / 8 * 8 * sh.row_tiles;
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
