// Microscaled 4-bit floating point (OCP MX, E2M1 elements under E8M0 scales of 32): quantisation and
// products (stt_mxfp4_* of include/stt_mi355x.h).
#include "stt_common.h"

typedef __bf16 mx_bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 mx_h2 __attribute__((ext_vector_type(2)));
typedef float mx_f4 __attribute__((ext_vector_type(4)));
typedef int mx_i8 __attribute__((ext_vector_type(8)));

namespace {

// ---------------------------------------------------------------------------------------------
// Quantisation.  Four neighbouring lanes own a block of 32: 8 elements each, the block's largest
// magnitude by two quad exchanges of its bit pattern (ordered like the magnitude, NaN on top).  With
// E its exponent field, floor(log2 max) - 2 + 127 = E - 2; below 2^-125 the scale stays at 2^-127.
// v_cvt_scalef32_pk_fp4_* divides by the scale (its exponent bits), rounds to nearest even and
// saturates at 6, two elements per instruction.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);
  v = v > a ? v : a;
  const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);
  return v > b ? v : b;
}

// scale byte of a block whose largest magnitude has the float32 bit pattern `top` (sign cleared)
__device__ __forceinline__ uint32_t block_scale(uint32_t top) {
  const uint32_t e = top >> 23;
  return e >= 255 ? 255u : e > 2 ? e - 2 : 0u;
}

__device__ __forceinline__ void load8(const float* x, float (&v)[8]) {
  const mx_f4 a = *(const mx_f4*)x, b = *(const mx_f4*)(x + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
__device__ __forceinline__ void load8(const _Float16* x, float (&v)[8]) {
  const uint4 u = *(const uint4*)x;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const mx_h2 h = __builtin_bit_cast(mx_h2, w[i]);
    v[2 * i] = (float)h[0]; v[2 * i + 1] = (float)h[1];
  }
}
__device__ __forceinline__ void load8(const __bf16* x, float (&v)[8]) {
  const uint4 u = *(const uint4*)x;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
}

template <typename T>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const T* x, long rows, long k8, long x_row, uint32_t* codes,
                                                             uint8_t* scales) {
  const long n = rows * k8;                    // k8 = eighths of a row; a multiple of 4, so quads never straddle rows
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long r = i / k8, c = i - r * k8;
    float v[8];
    load8(x + r * x_row + 8 * c, v);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t m = __float_as_uint(v[e]) & 0x7FFFFFFFu;
      top = top > m ? top : m;
    }
    const uint32_t s = block_scale(quad_max(top));
    const float scale = __uint_as_float(s << 23);
    uint32_t out = 0;
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[0], v[1], scale, 0);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[2], v[3], scale, 1);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[4], v[5], scale, 2);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[6], v[7], scale, 3);
    codes[i] = s == 255 ? 0u : out;
    if ((c & 3) == 0) scales[i >> 2] = (uint8_t)s;
  }
}

// two values of a code byte under the scale with exponent byte s (bits s << 23); exact in bf16
#define MX_PAIR(word, scale, sel) __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((word), (scale), (sel))

__device__ __forceinline__ uint4 expand8(uint32_t word, float scale) {
  uint4 u;
  u.x = __builtin_bit_cast(uint32_t, MX_PAIR(word, scale, 0));
  u.y = __builtin_bit_cast(uint32_t, MX_PAIR(word, scale, 1));
  u.z = __builtin_bit_cast(uint32_t, MX_PAIR(word, scale, 2));
  u.w = __builtin_bit_cast(uint32_t, MX_PAIR(word, scale, 3));
  return u;
}

template <bool F32>
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const uint32_t* codes, const uint8_t* scales, long n, void* out) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const uint4 u = expand8(codes[i], __uint_as_float((uint32_t)scales[i >> 2] << 23));
    if (!F32) {
      ((uint4*)out)[i] = u;
    } else {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
      float v[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(w[e] << 16); v[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u); }
      ((mx_f4*)out)[2 * i] = mx_f4{v[0], v[1], v[2], v[3]};
      ((mx_f4*)out)[2 * i + 1] = mx_f4{v[4], v[5], v[6], v[7]};
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Packed weights.  Tile (nt, kc) = rows 16 nt .. + 15, columns 128 kc .. + 127: lane l of a wave holds
// row l % 16 and the block of 32 columns l / 16 as 16 bytes of codes, which is the A operand of
// v_mfma_scale_f32_16x16x128_f8f6f4: [nt][kc][64 lanes][16 bytes].  Behind the codes the scales, one word
// per row and chunk with the scales of its four blocks: [nt][kc][16 rows].  Padding: codes 0, scale 1.
// ---------------------------------------------------------------------------------------------
struct Packed {
  long tiles_n, chunks;
  __host__ __device__ Packed(long n, long k) : tiles_n((n + 15) / 16), chunks((k + 127) / 128) {}
  __host__ __device__ long code_bytes() const { return tiles_n * chunks * 1024; }
  __host__ __device__ long scale_bytes() const { return tiles_n * chunks * 64; }
};

__global__ __launch_bounds__(256) void mxfp4_pack_kernel(const uint8_t* codes, const uint8_t* scales, long n, long k, uint4* out) {
  const Packed p(n, k);
  uint32_t* out_s = (uint32_t*)((uint8_t*)out + p.code_bytes());
  const long n_codes = p.tiles_n * p.chunks * 64, n_scales = p.tiles_n * p.chunks * 16;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n_codes + n_scales; i += (long)gridDim.x * 256) {
    if (i < n_codes) {
      const int lane = (int)(i & 63);
      const long kc = (i >> 6) % p.chunks, nt = (i >> 6) / p.chunks;
      const long row = nt * 16 + (lane & 15), col = kc * 128 + 32 * (lane >> 4);
      uint4 u = {0, 0, 0, 0};
      if (row < n && col < k) u = *(const uint4*)(codes + (row * k + col) / 2);
      out[i] = u;
    } else {
      const long j = i - n_codes;
      const long kc = (j >> 4) % p.chunks, row = (j >> 4) / p.chunks * 16 + (j & 15);
      uint32_t w = 0;
      for (int b = 0; b < 4; ++b) {
        const long col = kc * 128 + 32 * b;
        w |= (uint32_t)(row < n && col < k ? scales[(row * k + col) / 32] : 127) << (8 * b);
      }
      out_s[j] = w;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Epilogue of every product kernel: a lane holds n = n0 .. n0 + 3 of row m.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float gelu1(float v, int kind) {
  if (kind == STT_GELU_TANH) {
    const float c1 = -2.0f * 0.7978845608028654f * 1.4426950408889634f, c2 = c1 * 0.044715f;
    return v / (1.0f + __builtin_amdgcn_exp2f((v * v * c2 + c1) * v));
  }
  return kind == STT_GELU_ERF ? 0.5f * v * (1.0f + erff(v * 0.7071067811865476f)) : v;
}

__device__ __forceinline__ void store4(const stt_mxfp4_matmul_args& a, long m, long n0, mx_f4 v, bool vec) {
  if (m >= a.m || n0 >= a.n) return;
  const int nv = a.n - n0 < 4 ? (int)(a.n - n0) : 4;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (a.d_bias && r < nv) v[r] += a.d_bias[n0 + r];
    v[r] = gelu1(v[r], a.gelu);
  }
  const long at = m * a.out_row + n0;
  if (a.out_dtype == STT_F32) {
    float* o = (float*)a.d_out + at;
    if (vec && nv == 4) {
      if (a.accumulate) v += *(const mx_f4*)o;
      *(mx_f4*)o = v;
    } else {
      for (int r = 0; r < nv; ++r) o[r] = a.accumulate ? o[r] + v[r] : v[r];
    }
  } else {
    __bf16* o = (__bf16*)a.d_out + at;
    if (vec && nv == 4) {
      uint2 u;
      u.x = __builtin_bit_cast(uint32_t, mx_bf2{(__bf16)v[0], (__bf16)v[1]});
      u.y = __builtin_bit_cast(uint32_t, mx_bf2{(__bf16)v[2], (__bf16)v[3]});
      *(uint2*)o = u;
    } else {
      for (int r = 0; r < nv; ++r) o[r] = (__bf16)v[r];
    }
  }
}

// Lane group g of a wave (lanes 16 g ..) holds words d[i] = E[g][i]; afterwards d[i] = E[i][g].  Written as
// asm statements, since the swap builtins lose their second result in this compiler; the s_nop cover the
// wait states a swap needs after a vector instruction that wrote its operands.
__device__ __forceinline__ void transpose_groups(uint32_t (&d)[4]) {
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %2\n\tv_permlane32_swap_b32 %1, %3\n\ts_nop 1\n\t"
      "v_permlane16_swap_b32 %0, %1\n\tv_permlane16_swap_b32 %2, %3\n\ts_nop 1"
      : "+v"(d[0]), "+v"(d[1]), "+v"(d[2]), "+v"(d[3]));
}

// ---------------------------------------------------------------------------------------------
// Products.  A block owns 16 NT output features x 16 MT rows; its WK waves take the 128-column chunks of K
// round robin and their partial tiles are joined through LDS in wave order.  Weights come straight
// from memory in operand order (1 KiB per wave load), activations from the L2.  The weights are the A
// operand, so a lane ends up with 4 neighbouring features of one row.
//   bf16 activations: four v_mfma_f32_16x16x32_bf16 per chunk in the natural order of k (lane group g of
// step i: columns 32 i + 8 g ..), for which the weight words change lane groups (transpose_groups); codes
// become bf16 under their scale without rounding (v_cvt_scalef32_pk_bf16_fp4).
//   4-bit activations: one v_mfma_scale_f32_16x16x128_f8f6f4 per chunk.
// ---------------------------------------------------------------------------------------------
typedef uint32_t mx_u4 __attribute__((ext_vector_type(4)));

template <bool X4, int MT, int NT>
struct MxChunk {
  mx_u4 w[NT];
  uint32_t ws[NT];
  mx_u4 x[MT][X4 ? 1 : 4];
  uint32_t xs[X4 ? MT : 1];
};

// waves per SIMD whose registers (two sets of operands and the sums) fit
constexpr int mx_waves(bool x4, int mt, int nt) {
  return x4 ? (mt * nt >= 8 ? 2 : mt * nt >= 4 ? 3 : 4) : mt == 1 ? 4 : mt == 2 && nt <= 2 ? 3 : 2;
}

template <bool X4, int MT, int NT, int WK>
__global__ __launch_bounds__(64 * WK, mx_waves(X4, MT, NT)) void mxfp4_matmul_kernel(const stt_mxfp4_matmul_args a, int blocks_n, bool vec) {
  typedef MxChunk<X4, MT, NT> Chunk;
  const int tid = threadIdx.x, lane = tid & 63, wave = WK == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g = lane >> 4;
  const long bm = blockIdx.x / blocks_n, bn = blockIdx.x - bm * blocks_n;
  const Packed p(a.n, a.k);
  const int chunks = (int)p.chunks;
  // scalar bases, 32-bit lane offsets
  const uint8_t* wbase = (const uint8_t*)a.d_w;
  const uint8_t* sbase = wbase + p.code_bytes();
  const uint32_t woff = 16 * lane, soff = 4 * col;
  const long row_bytes = X4 ? a.k / 2 : 2 * a.x_row;
  const uint8_t* xbase = (const uint8_t*)a.d_x + bm * MT * 16 * row_bytes;
  const uint8_t* xsbase = X4 ? a.d_x_scales + bm * MT * 16 * (a.k / 32) : nullptr;
  uint32_t xoff[MT], xsoff[X4 ? MT : 1];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const long left = a.m - 1 - bm * MT * 16;
    const uint32_t r = t * 16 + col < left ? t * 16 + col : (uint32_t)left;
    xoff[t] = r * (uint32_t)row_bytes + 16 * g;
    if (X4) xsoff[X4 ? t : 0] = r * (uint32_t)(a.k / 32) + g;
  }
  mx_f4 acc[NT][MT];
#pragma unroll
  for (int u = 0; u < NT; ++u)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[u][t] = mx_f4{0.f, 0.f, 0.f, 0.f};

  auto load = [&](int c, Chunk& q) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const long nt = bn * NT + u < p.tiles_n ? bn * NT + u : p.tiles_n - 1;
      q.w[u] = *(const mx_u4*)(wbase + (nt * chunks + c) * 1024 + woff);
      q.ws[u] = *(const uint32_t*)(sbase + (nt * chunks + c) * 64 + soff);
    }
    const int left = (int)(a.k - (long)c * 128);        // columns from here on; uniform
    if (left >= 128) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (X4) {
          q.x[t][0] = *(const mx_u4*)(xbase + (long)c * 64 + xoff[t]);
          q.xs[X4 ? t : 0] = xsbase[c * 4 + xsoff[X4 ? t : 0]];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) q.x[t][X4 ? 0 : i] = *(const mx_u4*)(xbase + (long)c * 256 + 64 * i + xoff[t]);
        }
      }
    } else {                                           // the last chunk of a k that is not a multiple of 128
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (X4) {
          q.x[t][0] = mx_u4{0, 0, 0, 0};
          q.xs[X4 ? t : 0] = 127;
          if (32 * g < left) {
            q.x[t][0] = *(const mx_u4*)(xbase + (long)c * 64 + xoff[t]);
            q.xs[X4 ? t : 0] = xsbase[c * 4 + xsoff[X4 ? t : 0]];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            q.x[t][X4 ? 0 : i] = mx_u4{0, 0, 0, 0};
            if (32 * i < left) q.x[t][X4 ? 0 : i] = *(const mx_u4*)(xbase + (long)c * 256 + 64 * i + xoff[t]);
          }
        }
      }
    }
  };
  auto work = [&](const Chunk& q) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      if (X4) {
        const mx_i8 wa = {(int)q.w[u].x, (int)q.w[u].y, (int)q.w[u].z, (int)q.w[u].w, 0, 0, 0, 0};
        const int s = (int)((q.ws[u] >> (8 * g)) & 255u);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const mx_u4 xv = q.x[t][0];
          const mx_i8 xb = {(int)xv.x, (int)xv.y, (int)xv.z, (int)xv.w, 0, 0, 0, 0};
          acc[u][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xb, acc[u][t], 4, 4, 0, s, 0, (int)q.xs[X4 ? t : 0]);
        }
      } else {
        uint32_t d[4] = {q.w[u].x, q.w[u].y, q.w[u].z, q.w[u].w};
        transpose_groups(d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float scale = __uint_as_float(((q.ws[u] >> (8 * i)) & 255u) << 23);
          const mx_bf8 wf = __builtin_bit_cast(mx_bf8, expand8(d[i], scale));
#pragma unroll
          for (int t = 0; t < MT; ++t)
            acc[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, __builtin_bit_cast(mx_bf8, q.x[t][X4 ? 0 : i]), acc[u][t], 0, 0, 0);
        }
      }
    }
  };
  // two register sets alternate between "in flight" and "being used"
  Chunk qa, qb;
  if (wave < chunks) load(wave, qa);
  for (int c = wave; c < chunks; c += 2 * WK) {
    if (c + WK < chunks) load(c + WK, qb);
    work(qa);
    if (c + 2 * WK < chunks) load(c + 2 * WK, qa);
    if (c + WK < chunks) work(qb);
  }
  if (WK == 1) {
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int t = 0; t < MT; ++t) store4(a, (bm * MT + t) * 16 + col, (bn * NT + u) * 16 + 4 * g, acc[u][t], vec);
  } else {
    __shared__ mx_f4 part[WK][NT * MT][64];
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int t = 0; t < MT; ++t) part[wave][u * MT + t][lane] = acc[u][t];
    __syncthreads();
    for (int e = wave; e < NT * MT; e += WK) {
      mx_f4 v = part[0][e][lane];
#pragma unroll
      for (int w = 1; w < WK; ++w) v += part[w][e][lane];
      store4(a, (bm * MT + e % MT) * 16 + col, (bn * NT + e / MT) * 16 + 4 * g, v, vec);
    }
  }
}

unsigned grid_for(int64_t items) {
  const int64_t b = (items + 255) / 256;
  return (unsigned)(b < 1 ? 1 : b > 16384 ? 16384 : b);
}

// Tile and K split: MT from the rows; the widest NT, then the fewest waves along K, that still give
// kWaves waves (a chip's worth at two to four a SIMD), so that activations are read as few times as possible.
constexpr int64_t kWaves = 2048;
template <bool X4>
int launch_matmul(const stt_mxfp4_matmul_args& a, const Packed& p, bool vec, hipStream_t st) {
  const int64_t tiles_m = (a.m + 15) / 16;
  int mt = tiles_m == 1 ? 1 : tiles_m == 2 || !X4 ? 2 : 4, nt = mt == 1 ? 2 : 4, wk = 1;
  const int64_t bm = (tiles_m + mt - 1) / mt;
  auto waves = [&](int t) { return bm * ((p.tiles_n + t - 1) / t); };
  while (nt > 1 && waves(nt) * 8 < kWaves) nt >>= 1;
  while (wk < 8 && waves(nt) * wk < kWaves && wk * 2 <= p.chunks) wk <<= 1;
  const int64_t blocks_n = (p.tiles_n + nt - 1) / nt, blocks = bm * blocks_n;
  if (blocks > 0x7fffffff) return stt_fail(STT_ERR_UNSUPPORTED, "product of %lld x %lld", (long long)a.m, (long long)a.n);
#define STT_MM(MT, NT, WK)                                                                                               \
  if (mt == MT && nt == NT && wk == WK) {                                                                                \
    hipLaunchKernelGGL((mxfp4_matmul_kernel<X4, MT, NT, WK>), dim3((unsigned)blocks), dim3(64 * WK), 0, st, a, (int)blocks_n, vec); \
    return STT_OK;                                                                                                       \
  }
#define STT_MM_WK(MT, NT) if constexpr (X4 || MT <= 2) { STT_MM(MT, NT, 1) STT_MM(MT, NT, 2) STT_MM(MT, NT, 4) STT_MM(MT, NT, 8) }
  STT_MM_WK(1, 1) STT_MM_WK(1, 2) STT_MM_WK(2, 1) STT_MM_WK(2, 2) STT_MM_WK(2, 4) STT_MM_WK(4, 1) STT_MM_WK(4, 2) STT_MM_WK(4, 4)
#undef STT_MM_WK
#undef STT_MM
  return stt_fail(STT_ERR_UNSUPPORTED, "no kernel for tile %d x %d", mt, nt);
}

}  // namespace

extern "C" {

int stt_mxfp4_quantize(const void* d_x, int dtype, int64_t rows, int64_t k, int64_t x_row, uint8_t* d_codes,
                       uint8_t* d_scales, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (rows < 0 || k < 0 || k % 32) return stt_fail(STT_ERR_INVALID_ARGUMENT, "%lld rows of %lld: k must be a multiple of 32", (long long)rows, (long long)k);
  if (dtype != STT_F32 && dtype != STT_BF16 && dtype != STT_F16) return stt_fail(STT_ERR_UNSUPPORTED, "dtype %d", dtype);
  if (rows == 0 || k == 0) return STT_OK;
  if (!d_x || !d_codes || !d_scales) return stt_fail(STT_ERR_INVALID_ARGUMENT, "null argument");
  const int64_t unit = dtype == STT_F32 ? 4 : 8;
  if (((uintptr_t)d_x & 15) || ((uintptr_t)d_codes & 15) || (rows > 1 && (x_row < k || x_row % unit)))
    return stt_fail(STT_ERR_INVALID_ARGUMENT, "rows must be 16-byte aligned and at least k apart (row stride %lld)", (long long)x_row);
  const unsigned blocks = grid_for(rows * (k / 8));
#define STT_Q(T) hipLaunchKernelGGL(mxfp4_quantize_kernel<T>, dim3(blocks), dim3(256), 0, st, (const T*)d_x, (long)rows, (long)(k / 8), (long)x_row, (uint32_t*)d_codes, d_scales)
  if (dtype == STT_F32) STT_Q(float); else if (dtype == STT_BF16) STT_Q(__bf16); else STT_Q(_Float16);
#undef STT_Q
  STT_HIP_OR_FAIL(hipGetLastError(), (void)0);
  return STT_OK;
}

int stt_mxfp4_dequantize(const uint8_t* d_codes, const uint8_t* d_scales, int64_t rows, int64_t k, void* d_out,
                         int dtype, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (rows < 0 || k < 0 || k % 32) return stt_fail(STT_ERR_INVALID_ARGUMENT, "%lld rows of %lld: k must be a multiple of 32", (long long)rows, (long long)k);
  if (dtype != STT_F32 && dtype != STT_BF16) return stt_fail(STT_ERR_UNSUPPORTED, "dtype %d: STT_F32 or STT_BF16", dtype);
  if (rows == 0 || k == 0) return STT_OK;
  if (!d_codes || !d_scales || !d_out) return stt_fail(STT_ERR_INVALID_ARGUMENT, "null argument");
  if (((uintptr_t)d_codes & 15) || ((uintptr_t)d_out & 15)) return stt_fail(STT_ERR_INVALID_ARGUMENT, "pointers must be 16-byte aligned");
  const int64_t n = rows * (k / 8);
  if (dtype == STT_F32)
    hipLaunchKernelGGL(mxfp4_dequantize_kernel<true>, dim3(grid_for(n)), dim3(256), 0, st, (const uint32_t*)d_codes, d_scales, (long)n, d_out);
  else
    hipLaunchKernelGGL(mxfp4_dequantize_kernel<false>, dim3(grid_for(n)), dim3(256), 0, st, (const uint32_t*)d_codes, d_scales, (long)n, d_out);
  STT_HIP_OR_FAIL(hipGetLastError(), (void)0);
  return STT_OK;
}

size_t stt_mxfp4_packed_bytes(int64_t n, int64_t k) {
  if (n <= 0 || k <= 0) return 0;
  const Packed p(n, k);
  return (size_t)(p.code_bytes() + p.scale_bytes());
}

int stt_mxfp4_pack(const uint8_t* d_codes, const uint8_t* d_scales, int64_t n, int64_t k, void* d_packed, void* stream) {
  if (n < 0 || k < 0 || k % 32) return stt_fail(STT_ERR_INVALID_ARGUMENT, "%lld rows of %lld: k must be a multiple of 32", (long long)n, (long long)k);
  if (n == 0 || k == 0) return STT_OK;
  if (!d_codes || !d_scales || !d_packed) return stt_fail(STT_ERR_INVALID_ARGUMENT, "null argument");
  if (((uintptr_t)d_codes & 15) || ((uintptr_t)d_packed & 15)) return stt_fail(STT_ERR_INVALID_ARGUMENT, "pointers must be 16-byte aligned");
  const Packed p(n, k);
  hipLaunchKernelGGL(mxfp4_pack_kernel, dim3(grid_for(p.tiles_n * p.chunks * 80)), dim3(256), 0, (hipStream_t)stream,
                     d_codes, d_scales, (long)n, (long)k, (uint4*)d_packed);
  STT_HIP_OR_FAIL(hipGetLastError(), (void)0);
  return STT_OK;
}

int stt_mxfp4_matmul(const stt_mxfp4_matmul_args* a, void* stream) {
  hipStream_t st = (hipStream_t)stream;
  if (!a) return stt_fail(STT_ERR_INVALID_ARGUMENT, "null argument");
  if (a->m < 0 || a->n < 0 || a->k < 32 || a->k % 32)
    return stt_fail(STT_ERR_INVALID_ARGUMENT, "product of %lld x %lld x %lld: k must be a positive multiple of 32",
                    (long long)a->m, (long long)a->n, (long long)a->k);
  if (a->out_dtype != STT_F32 && a->out_dtype != STT_BF16) return stt_fail(STT_ERR_UNSUPPORTED, "output dtype %d: STT_F32 or STT_BF16", a->out_dtype);
  if (a->gelu < STT_GELU_NONE || a->gelu > STT_GELU_ERF) return stt_fail(STT_ERR_UNSUPPORTED, "gelu %d", a->gelu);
  if (a->accumulate && (a->out_dtype != STT_F32 || a->gelu))
    return stt_fail(STT_ERR_UNSUPPORTED, "accumulation needs an STT_F32 output and no GELU");
  if (a->m == 0 || a->n == 0) return STT_OK;
  if (!a->d_x || !a->d_w || !a->d_out) return stt_fail(STT_ERR_INVALID_ARGUMENT, "null argument");
  if (((uintptr_t)a->d_x & 15) || ((uintptr_t)a->d_w & 15)) return stt_fail(STT_ERR_INVALID_ARGUMENT, "pointers must be 16-byte aligned");
  if (!a->d_x_scales && a->m > 1 && (a->x_row < a->k || a->x_row % 8))
    return stt_fail(STT_ERR_INVALID_ARGUMENT, "row stride %lld: at least k, a multiple of 8", (long long)a->x_row);
  if (a->k >= 1 << 25 || (!a->d_x_scales && a->m > 1 && a->x_row >= 1 << 25))
    return stt_fail(STT_ERR_UNSUPPORTED, "rows of 2^25 elements and more");
  if (a->m > 1 && a->out_row < a->n) return stt_fail(STT_ERR_INVALID_ARGUMENT, "output row stride %lld below n", (long long)a->out_row);
  const Packed p(a->n, a->k);
  // 4 outputs of a lane go out in one store where every group of 4 is aligned to its size
  const int size = a->out_dtype == STT_F32 ? 16 : 8;
  const bool vec = ((uintptr_t)a->d_out % size) == 0 && a->out_row % 4 == 0;
  const int rc = a->d_x_scales ? launch_matmul<true>(*a, p, vec, st) : launch_matmul<false>(*a, p, vec, st);
  if (rc) return rc;
  STT_HIP_OR_FAIL(hipGetLastError(), (void)0);
  return STT_OK;
}

}  // extern "C"
