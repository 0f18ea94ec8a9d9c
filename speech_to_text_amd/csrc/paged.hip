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
constexpr int kPlanPer = STT_PLAN_MAX_REQUESTS / kPlanThreads;

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

  // this thread's run of consecutive requests
  long long own[3] = {0, 0, 0};
  int bad = 0;                                 // bit 0: state, bit 1: too long
  int take[kPlanPer], give[kPlanPer], fresh[kPlanPer];
#pragma unroll
  for (int u = 0; u < kPlanPer; ++u) {
    const int i = tid * per + u;
    take[u] = give[u] = fresh[u] = 0;
    if (u < per && i < a.n) {
      const int c = a.cached[i], w = a.fresh[i], h = a.held_in[i];
      if (c < 0 || w < 0 || h < 0 || h > a.width) bad |= 1;
      const long long need = ((long long)c + w + ((1LL << a.shift) - 1)) >> a.shift;
      if (need > a.width) bad |= 2;
      if (!bad) {
        const int d = (int)need - h;
        take[u] = d > 0 ? d : 0;
        give[u] = d < 0 ? -d : 0;
        fresh[u] = w;
      }
    }
    own[0] += take[u]; own[1] += give[u]; own[2] += fresh[u];
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
#pragma unroll
  for (int u = 0; u < kPlanPer; ++u) {
    const int i = tid * per + u;
    if (u < per && i < a.n) {
      s_take[i] = (int)before[0]; s_give[i] = (int)before[1]; s_start[i] = (int)before[2];
    }
    before[0] += take[u]; before[1] += give[u]; before[2] += fresh[u];
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
// Tree attention.  One wave per (node, head): the wave walks the keys 64 at a time, a lane scores one
// key, the running maximum and sum of the softmax follow the tiles, then the lanes turn to the
// features for the weighted sum.
// ---------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f32(half_bits v);
template <> __device__ __forceinline__ float to_f32<__bf16>(half_bits v) { return __uint_as_float((uint32_t)v << 16); }
template <> __device__ __forceinline__ float to_f32<_Float16>(half_bits v) { return (float)__builtin_bit_cast(_Float16, v); }

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

template <typename T, int D>
__global__ __launch_bounds__(64) void tree_attention_plain_kernel(const stt_tree_attention_args a) {
  __shared__ float qs[D];
  __shared__ float ps[64];
  const int lane = threadIdx.x;
  long id = blockIdx.x;
  const int node = (int)(id % a.max_nodes);
  id /= a.max_nodes;
  const int h = (int)(id % a.n_heads), seq = (int)(id / a.n_heads);
  const int row0 = a.d_starts[seq];
  int nodes = a.d_starts[seq + 1] - row0;
  nodes = nodes < a.max_nodes ? nodes : a.max_nodes;
  if (node >= nodes || row0 < 0 || row0 + nodes > a.rows) return;
  const int group = a.n_heads / a.n_kv_heads, hk = h / group;
  const unsigned long long path = __shfl(tree_path(a.d_parents, row0, nodes, lane), node, 64);
  const half_bits* q = (const half_bits*)a.d_q + (row0 + node) * a.q_row + h * a.q_head;
  for (int e = lane; e < D; e += 64) qs[e] = to_f32<T>(q[e]) * (a.scale * 1.4426950408889634f);
  __syncthreads();
  int cached = a.d_cached[seq];
  const long most = (long)a.width * a.block_size;
  cached = cached < 0 ? 0 : cached < most ? cached : (int)most;
  const int shift = __builtin_ctz(a.block_size);
  const half_bits* kc = (const half_bits*)a.d_k_cache + hk * a.head_stride;
  const half_bits* vc = (const half_bits*)a.d_v_cache + hk * a.head_stride;
  const half_bits* kn = (const half_bits*)a.d_k + row0 * a.k_row + hk * a.k_head;
  const half_bits* vn = (const half_bits*)a.d_v + row0 * a.v_row + hk * a.v_head;
  float m = -__builtin_inff(), sum = 0.f, acc[D / 64];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) acc[e] = 0.f;
  for (long k0 = 0; k0 < (long)cached + nodes; k0 += 64) {
    const long key = k0 + lane;
    const half_bits* kp = nullptr;
    long vat = -1;                              // >= 0: offset in the cache; < 0: -1 - offset in the new rows
    if (key < cached) {
      const int b = a.d_table[(long)seq * a.width + (key >> shift)];
      if (b >= 0 && b < a.n_blocks) {
        vat = b * a.block_stride + (key & (a.block_size - 1)) * a.pos_stride;
        kp = kc + vat;
      }
    } else if (key < cached + nodes && ((path >> (key - cached)) & 1)) {
      kp = kn + (key - cached) * a.k_row;
      vat = -1 - (key - cached) * a.v_row;
    }
    float s = -__builtin_inff();
    if (kp) {
      s = 0.f;
#pragma unroll
      for (int e = 0; e < D; e += 8) {
        const uint4 u = *(const uint4*)(kp + e);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s += qs[e + 2 * j] * to_f32<T>((half_bits)(w[j] & 0xFFFF));
          s += qs[e + 2 * j + 1] * to_f32<T>((half_bits)(w[j] >> 16));
        }
      }
    }
    float top = s;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float mn = fmaxf(m, top);
    const float ref = mn == -__builtin_inff() ? 0.f : mn;
    const float p = kp ? __builtin_amdgcn_exp2f(s - ref) : 0.f;
    const float keep = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    float ts = p;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ts += __shfl_xor(ts, o, 64);
    sum = sum * keep + ts;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) acc[e] *= keep;
    const unsigned long long live = __ballot(kp != nullptr);
    for (int j = 0; j < 64; ++j) {
      if (!((live >> j) & 1)) continue;
      const float pj = __shfl(p, j, 64);
      const long at = __shfl(vat, j, 64);
      const half_bits* vp = at >= 0 ? vc + at : vn + (-1 - at);
#pragma unroll
      for (int e = 0; e < D / 64; ++e) acc[e] += pj * to_f32<T>(vp[lane + 64 * e]);
    }
  }
  half_bits* out = (half_bits*)a.d_out + (row0 + node) * a.out_row + h * a.out_head;
#pragma unroll
  for (int e = 0; e < D / 64; ++e) out[lane + 64 * e] = __builtin_bit_cast(half_bits, (T)(acc[e] / sum));
  if (h % group == 0) {                         // store the node's K/V, once per KV head
    const long slot = a.d_slots[row0 + node];
    if (slot >= 0 && slot < (long)a.n_blocks * a.block_size) {
      const long at = (slot >> shift) * a.block_stride + hk * a.head_stride + (slot & (a.block_size - 1)) * a.pos_stride;
#pragma unroll
      for (int e = 0; e < D; e += 64) {
        ((half_bits*)a.d_k_cache)[at + lane + e] = kn[node * a.k_row + lane + e];
        ((half_bits*)a.d_v_cache)[at + lane + e] = vn[node * a.v_row + lane + e];
      }
    }
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

size_t stt_tree_attention_workspace_bytes(const stt_tree_attention_args* args) { (void)args; return 0; }

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
  const int64_t blocks = (int64_t)a->n_seq * a->n_heads * a->max_nodes;
  if (blocks > 0x7fffffff) return stt_fail(STT_ERR_UNSUPPORTED, "%lld blocks", (long long)blocks);
#define STT_TREE(T, D) hipLaunchKernelGGL((tree_attention_plain_kernel<T, D>), dim3((unsigned)blocks), dim3(64), 0, st, *a)
  if (a->dtype == STT_BF16) { if (a->head_dim == 64) STT_TREE(__bf16, 64); else STT_TREE(__bf16, 128); }
  else { if (a->head_dim == 64) STT_TREE(_Float16, 64); else STT_TREE(_Float16, 128); }
#undef STT_TREE
  STT_HIP_OR_FAIL(hipGetLastError(), (void)0);
  return STT_OK;
}

}  // extern "C"
