// Microscaled 4-bit floating point (OCP MX, E2M1 elements under E8M0 scales of 32): quantisation and
// products (stt_mxfp4_* of include/stt_mi355x.h).
#include <type_traits>

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
// saturates at 6, two elements per instruction.  Bound by HBM: 51 866 x 1 280 float32 (265 MB in, 35 out)
// 61 us, back to bf16 25 us; 9 x 1 280 2.4 us, a launch.
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
template <int KIND>
__device__ __forceinline__ float gelu1(float v) {
  if (KIND == STT_GELU_TANH) {
    const float c1 = -2.0f * 0.7978845608028654f * 1.4426950408889634f, c2 = c1 * 0.044715f;
    // (exponential and reciprocal to one unit in the last place, off by 1.8 x 2^-24 |v| at most together, and without
    // the cancellation of 1 + tanh for negative v; an overflowing exponential gives v * 0)
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f((v * v * c2 + c1) * v));
  }
  return KIND == STT_GELU_ERF ? 0.5f * v * (1.0f + erff(v * 0.7071067811865476f)) : v;
}

// what is added to features n0 .. n0 + 3 (features past the end read the last one: never stored)
__device__ __forceinline__ mx_f4 bias4(const stt_mxfp4_matmul_args& a, const float* bias, long n0) {
  mx_f4 b;
#pragma unroll
  for (int r = 0; r < 4; ++r) b[r] = bias[n0 + r < a.n ? n0 + r : a.n - 1];
  return b;
}

template <int GELU, bool F32>
__device__ __forceinline__ void store4(const stt_mxfp4_matmul_args& a, long m, long n0, mx_f4 v, mx_f4 bias, bool vec) {
  if (m >= a.m || n0 >= a.n) return;
  const int nv = a.n - n0 < 4 ? (int)(a.n - n0) : 4;
  v += bias;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = gelu1<GELU>(v[r]);
  const long at = m * a.out_row + n0;
  if (F32) {
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

// f(store) with the store of the call's activation and output type; the choice is uniform
template <typename F>
__device__ __forceinline__ void with_store(const stt_mxfp4_matmul_args& a, bool vec, F f) {
#define STT_CASE(GELU, F32) \
  f([&](long m, long n0, mx_f4 v, mx_f4 b) __attribute__((always_inline)) { store4<GELU, F32>(a, m, n0, v, b, vec); })
  if (a.out_dtype == STT_F32) {
    if (a.gelu == STT_GELU_NONE) STT_CASE(STT_GELU_NONE, true);
    else if (a.gelu == STT_GELU_TANH) STT_CASE(STT_GELU_TANH, true);
    else STT_CASE(STT_GELU_ERF, true);
  } else {
    if (a.gelu == STT_GELU_NONE) STT_CASE(STT_GELU_NONE, false);
    else if (a.gelu == STT_GELU_TANH) STT_CASE(STT_GELU_TANH, false);
    else STT_CASE(STT_GELU_ERF, false);
  }
#undef STT_CASE
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
// Few rows are bound by the weights' bytes and a block's start-up: 1 x 5 120 x 1 280 3.8 us, 9 x 51 866 x 1 280 with
// float32 output (37 MB) 11 us.  Some hundred rows by what the blocks read from the L2: 600 x 1 280 x 5 120 27 us.
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

  auto load_w = [&](int c, Chunk& q) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const long nt = bn * NT + u < p.tiles_n ? bn * NT + u : p.tiles_n - 1;
      q.w[u] = *(const mx_u4*)(wbase + (nt * chunks + c) * 1024 + woff);
      q.ws[u] = *(const uint32_t*)(sbase + (nt * chunks + c) * 64 + soff);
    }
  };
  auto load = [&](int c, Chunk& q) __attribute__((always_inline)) {
    load_w(c, q);
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
  };
  // the last chunk of a k that is not a multiple of 128: nothing is read past the rows' ends
  auto load_tail = [&](int c, Chunk& q) __attribute__((always_inline)) {
    const int left = (int)(a.k - (long)c * 128);
    load_w(c, q);
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
  // Two register sets alternate between "in flight" and "being used"; chunks past the end are fetched as the
  // last one again (a branch around a load makes the compiler wait for everything in flight).
  const int full = (int)(a.k / 128);
  auto within = [&](int c) __attribute__((always_inline)) { return c < full ? c : full - 1; };
  Chunk qa, qb;
  if (wave < full) {
    load(wave, qa);
    int c = wave;
    for (; c + WK < full; c += 2 * WK) {
      load(c + WK, qb);
      work(qa);
      load(within(c + 2 * WK), qa);
      work(qb);
    }
    if (c < full) work(qa);
  }
  if (full < chunks && wave == full % WK) {
    load_tail(full, qa);
    work(qa);
  }
  if (WK == 1) {
    with_store(a, vec, [&](auto store) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const mx_f4 b = a.d_bias ? bias4(a, a.d_bias, (bn * NT + u) * 16 + 4 * g) : mx_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < MT; ++t) store((bm * MT + t) * 16 + col, (bn * NT + u) * 16 + 4 * g, acc[u][t], b);
      }
    });
  } else {
    __shared__ mx_f4 part[WK][NT * MT][64];
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int t = 0; t < MT; ++t) part[wave][u * MT + t][lane] = acc[u][t];
    __syncthreads();
    for (int e = wave; e < NT * MT; e += WK) {
      const long m = (bm * MT + e % MT) * 16 + col, n0 = (bn * NT + e / MT) * 16 + 4 * g;
      const mx_f4 b = a.d_bias ? bias4(a, a.d_bias, n0) : mx_f4{0.f, 0.f, 0.f, 0.f};
      mx_f4 v = part[0][e][lane];
#pragma unroll
      for (int w = 1; w < WK; ++w) v += part[w][e][lane];
      with_store(a, vec, [&](auto store) __attribute__((always_inline)) { store(m, n0, v, b); });
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Many rows: a block of four waves owns 128 rows x 256 or 128 features (a wave a quarter) and takes K in chunks of 128
// through LDS, two stages: while chunk c is multiplied, chunk c + 1 goes from registers to the other stage
// and chunk c + 2 is on its way to registers; one barrier a chunk.  Operands lie in LDS in
// fragment order, permuted against bank conflicts (fragment_slot).  blockIdx % 8 picks the XCD; it takes
// kBigGroup row tiles at a time through the feature tiles, so that what its blocks read at one time fits
// its L2.  A last chunk of fewer columns follows by itself: what lies behind a row's end is read inside the
// row instead and goes to LDS as zeros.  (K below 128 takes the kernel above.)
//   4-bit activations: v_mfma_scale_f32_32x32x64_f8f6f4, two per chunk and 32 x 32 tile.  (Alone on the chip
// it reaches 7.1 PFLOP/s here, the 16 x 16 x 128 form 4.7.)  A row's four scales are one word: shifted by
// the lane's block once, the instruction's byte select then picks between the two steps.
//   bf16 activations: v_mfma_f32_16x16x32_bf16; the weights, an eighth of the bytes, skip LDS.
// 24 000 x 5 120 x 1 280, 4-bit x 4-bit, GELU, bf16 out: 150 us (2.1 PFLOP/s), of which 45 are the 245 MB of
// output; bf16 activations reach 1.1 PFLOP/s.
// The tile leaves through LDS: a lane holds 4 neighbouring features, which would go out in pieces of 16 to
// 32 bytes a row; from LDS every row goes out in 128-byte runs, element by element where rows are not 16-byte
// aligned (13 737 x 9 127 x 416 bf16 200 us, 285 in pieces of up to 8 bytes).
// ---------------------------------------------------------------------------------------------
typedef float mx_f16 __attribute__((ext_vector_type(16)));
constexpr int kBigGroup = 8;
struct __attribute__((packed)) Unaligned32 { uint32_t v; };
template <bool X4> constexpr int kBigFeatures = X4 ? 256 : 128;

// Place of (row, lane group) of a 16-row fragment in its 1 KiB.  The exclusive or spreads the writes, which
// come row by row (4 pieces a row, 16 for `step`), over the banks and keeps the reads of a fragment apart.
__device__ __forceinline__ int fragment_slot(int row, int g, int step) {
  return g * 16 + (row ^ ((g & 1) * 12) ^ ((g >> 1) * 4) ^ step);
}

template <bool X4>
__global__ __launch_bounds__(256, 2) void mxfp4_matmul_big_kernel(const stt_mxfp4_matmul_args a, int tiles_m, int tiles_n, bool vec16) {
  constexpr int BM = 128, BN = kBigFeatures<X4>, MT = X4 ? 2 : 4, TILE = X4 ? 32 : 16, NT = BN / 2 / TILE;
  constexpr int XB = X4 ? BM * 64 : BM * 256;          // bytes of activations per chunk
  constexpr int WB = X4 ? BN * 64 : 0;                 // ... of weights that go through LDS
  constexpr int SB = X4 ? BM * 4 : 0;                  // ... of activation scales
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][XB + WB + SB];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & (TILE - 1), g = lane / TILE, wm = wave & 1, wn = wave >> 1;
  // an eighth of the tiles per XCD, in one order: kBigGroup row tiles side by side, feature tile after feature tile
  const int tiles = tiles_m * tiles_n, per = (tiles + 7) >> 3, order = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || order >= tiles) return;
  const int group = order / (kBigGroup * tiles_n), in = order - group * (kBigGroup * tiles_n);
  const int high = tiles_m - group * kBigGroup < kBigGroup ? tiles_m - group * kBigGroup : kBigGroup;
  const int tm = group * kBigGroup + in % high, tn = in / high;
  const Packed p(a.n, a.k);
  const int chunks = (int)p.chunks, full = (int)(a.k >> 7);      // (full >= 1)
  const long m0 = (long)tm * BM, nt0 = (long)tn * (BN / 16);
  const uint8_t* wcodes = (const uint8_t*)a.d_w;
  const uint8_t* wscales = wcodes + p.code_bytes();

  // staging: what this thread fetches of a chunk
  constexpr int XN = XB / 16 / 256, WN = WB / 16 / 256;
  struct Fetched { mx_u4 x[XN], w[X4 ? WN : 1]; uint32_t s; } fa;
  constexpr int PIECES = X4 ? 4 : 16;                  // 16-byte pieces of a row in a chunk
  const long row_bytes = X4 ? a.k / 2 : 2 * a.x_row;
  const uint8_t* xbase = (const uint8_t*)a.d_x + m0 * row_bytes;
  uint32_t xoff[XN];                                   // (128 rows span less than 2^32 bytes: checked)
#pragma unroll
  for (int i = 0; i < XN; ++i) {
    const int at = tid + 256 * i;
    const long left = a.m - 1 - m0;
    const uint32_t r = at / PIECES < left ? at / PIECES : (uint32_t)left;
    xoff[i] = r * (uint32_t)row_bytes + 16 * (at % PIECES);
  }
  const uint8_t* xsp = nullptr;
  long wtile[X4 ? WN : 1];
  if (X4) {
    const long m = m0 + (tid & (BM - 1));
    xsp = a.d_x_scales + (m < a.m ? m : a.m - 1) * (a.k / 32);
#pragma unroll
    for (int i = 0; i < WN; ++i) {
      const long nt = nt0 + (tid >> 6) + 4 * i;
      wtile[X4 ? i : 0] = (nt < p.tiles_n ? nt : p.tiles_n - 1) * chunks * 1024;
    }
  }
  auto fetch = [&](int c, Fetched& f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < XN; ++i) f.x[i] = *(const mx_u4*)(xbase + (long)c * (16 * PIECES) + xoff[i]);
    if (X4) {
#pragma unroll
      for (int i = 0; i < WN; ++i) f.w[X4 ? i : 0] = *(const mx_u4*)(wcodes + wtile[X4 ? i : 0] + c * 1024 + 16 * lane);
      f.s = ((const Unaligned32*)(xsp + 4 * c))->v;      // (rows of k / 32 bytes)
    }
  };
  auto put = [&](uint8_t* stage, const Fetched& f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < XN; ++i) {
      const int at = tid + 256 * i, row = at / PIECES, piece = at % PIECES, pg = piece & 3, step = piece >> 2;
      *(mx_u4*)(stage + ((row >> 4) * (PIECES / 4) + step) * 1024 + fragment_slot(row & 15, pg, step) * 16) = f.x[i];
    }
    if (X4) {
#pragma unroll
      for (int i = 0; i < WN; ++i) *(mx_u4*)(stage + XB + ((tid >> 6) + 4 * i) * 1024 + 16 * lane) = f.w[X4 ? i : 0];
      *(uint32_t*)(stage + XB + WB + 4 * (tid & (BM - 1))) = f.s;        // (two threads, the same word)
    }
  };
  // operands that go from memory to registers, one chunk ahead: scales, and the codes of the bf16 form
  struct Direct { mx_u4 w[X4 ? 1 : NT]; uint32_t s[NT]; } da, db;
  const uint8_t* dsp[NT];
  const uint8_t* dwp[X4 ? 1 : NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    long nt = X4 ? nt0 + (wn * NT + u) * 2 + (col >> 4) : nt0 + wn * NT + u;
    nt = nt < p.tiles_n ? nt : p.tiles_n - 1;
    dsp[u] = wscales + nt * chunks * 64 + 4 * (col & 15);
    if (!X4) dwp[X4 ? 0 : u] = wcodes + nt * chunks * 1024 + 16 * lane;
  }
  auto direct = [&](int c, Direct& q) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      q.s[u] = *(const uint32_t*)(dsp[u] + c * 64);
      if (!X4) q.w[X4 ? 0 : u] = *(const mx_u4*)(dwp[X4 ? 0 : u] + (long)c * 1024);
    }
  };
  typedef std::conditional_t<X4, mx_f16, mx_f4> Acc;
  Acc acc[NT][MT];
  // the sums start from the bias
  if (a.d_bias && nt0 * 16 + BN <= a.n && ((uintptr_t)a.d_bias & 15) == 0) {
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int q = 0; q < (X4 ? 4 : 1); ++q) {
        const mx_f4 v = *(const mx_f4*)(a.d_bias + nt0 * 16 + (wn * NT + u) * TILE + (X4 ? 8 * q : 0) + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[u][0][4 * q + r] = v[r];
      }
  } else if (a.d_bias) {
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int q = 0; q < (X4 ? 4 : 1); ++q) {
        const mx_f4 v = bias4(a, a.d_bias, nt0 * 16 + (wn * NT + u) * TILE + (X4 ? 8 * q : 0) + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[u][0][4 * q + r] = v[r];
      }
  } else {
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[u][0] = Acc{};
  }
#pragma unroll
  for (int u = 0; u < NT; ++u)
#pragma unroll
    for (int t = 1; t < MT; ++t) acc[u][t] = acc[u][0];

  // Chunks past the end are fetched as the last one again: with a branch around a load the compiler has to
  // assume the worst about what is in flight and waits for all of it.
  auto within = [&](int c) __attribute__((always_inline)) { return c < full ? c : full - 1; };
  fetch(0, fa);
  direct(0, da);
  put(lds[0], fa);
  fetch(within(1), fa);
  auto multiply = [&](const uint8_t* stage, const Direct& q) __attribute__((always_inline)) {
    if constexpr (X4) {
      uint32_t xs[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) xs[t] = *(const uint32_t*)(stage + XB + WB + ((wm * MT + t) * 32 + col) * 4) >> (8 * g);
#define STT_STEP(S)                                                                                                        \
  {                                                                                                                        \
    mx_u4 xf[MT], wf[NT];                                                                                                  \
    for (int t = 0; t < MT; ++t)                                                                                           \
      xf[t] = *(const mx_u4*)(stage + ((wm * MT + t) * 2 + (col >> 4)) * 1024 + fragment_slot(col & 15, 2 * S + g, 0) * 16); \
    for (int u = 0; u < NT; ++u)                                                                                           \
      wf[u] = *(const mx_u4*)(stage + XB + ((wn * NT + u) * 2 + (col >> 4)) * 1024 + ((2 * S + g) * 16 + (col & 15)) * 16);  \
    for (int u = 0; u < NT; ++u) {                                                                                         \
      const mx_i8 wa = {(int)wf[u].x, (int)wf[u].y, (int)wf[u].z, (int)wf[u].w, 0, 0, 0, 0};                               \
      const int ws = (int)(q.s[u] >> (8 * g));                                                                             \
      for (int t = 0; t < MT; ++t) {                                                                                       \
        const mx_i8 xb = {(int)xf[t].x, (int)xf[t].y, (int)xf[t].z, (int)xf[t].w, 0, 0, 0, 0};                             \
        acc[u][t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, xb, acc[u][t], 4, 4, 2 * S, ws, 2 * S, (int)xs[t]);  \
      }                                                                                                                    \
    }                                                                                                                      \
  }
      STT_STEP(0)
      STT_STEP(1)
#undef STT_STEP
    } else {
      uint32_t d[NT][4];
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const mx_u4 w = q.w[X4 ? 0 : u];
        d[u][0] = w.x; d[u][1] = w.y; d[u][2] = w.z; d[u][3] = w.w;
        transpose_groups(d[u]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mx_bf8 xf[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t)
          xf[t] = __builtin_bit_cast(mx_bf8, *(const mx_u4*)(stage + ((wm * MT + t) * 4 + i) * 1024 + fragment_slot(col, g, i) * 16));
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const mx_bf8 wf = __builtin_bit_cast(mx_bf8, expand8(d[u][i], __uint_as_float(((q.s[u] >> (8 * i)) & 255u) << 23)));
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[t], acc[u][t], 0, 0, 0);
        }
      }
    }
  };
  // chunk c from stage `at` and `q`; fa holds chunk c + 1 and then takes chunk c + 2, `ahead` takes chunk c + 1
  auto step = [&](int c, int at, const Direct& q, Direct& ahead) __attribute__((always_inline)) {
    direct(within(c + 1), ahead);
    lds_barrier();                                     // stage c is written, stage c - 1 is read
    put(lds[1 - at], fa);
    fetch(within(c + 2), fa);
    multiply(lds[at], q);
  };
  int c = 0;
  for (; c + 1 < full; c += 2) {
    step(c, 0, da, db);
    step(c + 1, 1, db, da);
  }
  if (c < full) step(c, 0, da, db);
  if (full < chunks) {                                 // 32, 64 or 96 columns more
    const int row_end = X4 ? (int)(a.k / 2) : 2 * (int)a.k, column = full * 16 * PIECES + 16 * (tid % PIECES);
    const bool beyond = column >= row_end;
    const uint32_t back = beyond ? (uint32_t)(column + 16 - row_end) : 0u;
#pragma unroll
    for (int i = 0; i < XN; ++i) {
      fa.x[i] = *(const mx_u4*)(xbase + (long)full * (16 * PIECES) + (long)xoff[i] - back);
      if (beyond) fa.x[i] = mx_u4{0, 0, 0, 0};
    }
    if (X4) {
#pragma unroll
      for (int i = 0; i < WN; ++i) fa.w[X4 ? i : 0] = *(const mx_u4*)(wcodes + wtile[X4 ? i : 0] + full * 1024 + 16 * lane);
      const int missing = 4 * chunks - (int)(a.k / 32);               // the row's last four scales, shifted into place
      fa.s = ((const Unaligned32*)(xsp + 4 * full - missing))->v >> (8 * missing);
    }
    direct(full, da);
    lds_barrier();                                     // the stages are read
    put(lds[0], fa);
    lds_barrier();
    multiply(lds[0], da);
  }

  const long mw = m0 + wm * 64, nw = nt0 * 16 + wn * (BN / 2);
  const bool whole = vec16 && nw + BN / 2 <= a.n;      // else an edge, or rows that are not 16-byte aligned
  __syncthreads();                                     // everybody is done with the stages
  // 64 rows of 128 bytes per wave, 16-byte piece p of row r at p ^ (r & 7): 64 bf16 features, or 32 float ones at a time
  uint8_t* mine = &lds[0][0] + wave * 8192;
  const int rr = lane >> 3, pp = lane & 7;
  auto flush = [&](int first, auto element) __attribute__((always_inline)) {     // from feature `first` on
    typedef decltype(element) E;
    typedef E __attribute__((may_alias)) Stored;       // (written as other types)
    constexpr int SIZE = sizeof(E), PER = 128 / SIZE;
    if (whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 8 * i + rr;
        mx_u4 v = *(const mx_u4*)(mine + r * 128 + ((pp ^ (r & 7)) * 16));
        if (mw + r < a.m) {
          uint8_t* o = (uint8_t*)a.d_out + ((mw + r) * a.out_row + nw + first) * SIZE + 16 * pp;
          if (a.accumulate) *(mx_f4*)o += __builtin_bit_cast(mx_f4, v);
          else *(mx_u4*)o = v;
        }
      }
      return;
    }
    // one element a lane: still 128 bytes of a row side by side
    const int f = lane % PER, p16 = f * SIZE / 16;
    if (nw + first + f >= a.n) return;
#pragma unroll 8
    for (int r = lane / PER; r < 64; r += 64 / PER) {
      const E v = *(const Stored*)(mine + r * 128 + ((p16 ^ (r & 7)) * 16) + f * SIZE % 16);
      if (mw + r >= a.m) break;
      E* o = (E*)a.d_out + (mw + r) * a.out_row + nw + first + f;
      if (SIZE == 4 && a.accumulate) *(float*)o += __builtin_bit_cast(float, (uint32_t)v);
      else *o = v;
    }
  };
  auto leave = [&](auto act) __attribute__((always_inline)) {
    if (a.out_dtype == STT_BF16) {
      constexpr int PER = 64 / TILE;                   // tiles whose features fill 128 bytes of a row
#pragma unroll
      for (int u0 = 0; u0 < NT; u0 += PER) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int u = u0; u < u0 + PER; ++u)
#pragma unroll
            for (int q = 0; q < (X4 ? 4 : 1); ++q) {
              const int r = t * TILE + col, f = (u - u0) * TILE + (X4 ? 8 * q : 0) + 4 * g;
              const uint32_t lo = __builtin_bit_cast(uint32_t, mx_bf2{(__bf16)act(acc[u][t][4 * q]), (__bf16)act(acc[u][t][4 * q + 1])});
              const uint32_t hi = __builtin_bit_cast(uint32_t, mx_bf2{(__bf16)act(acc[u][t][4 * q + 2]), (__bf16)act(acc[u][t][4 * q + 3])});
              *(uint2*)(mine + r * 128 + (((f >> 3) ^ (r & 7)) * 16) + (f & 4) * 2) = uint2{lo, hi};
            }
        flush(u0 * TILE, (uint16_t)0);
      }
    } else {
      constexpr int PER = 32 / TILE;
#pragma unroll
      for (int u0 = 0; u0 < NT; u0 += PER) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int u = u0; u < u0 + PER; ++u)
#pragma unroll
            for (int q = 0; q < (X4 ? 4 : 1); ++q) {
              const int r = t * TILE + col, f = (u - u0) * TILE + (X4 ? 8 * q : 0) + 4 * g;
              *(mx_f4*)(mine + r * 128 + (((f >> 2) ^ (r & 7)) * 16)) =
                  mx_f4{act(acc[u][t][4 * q]), act(acc[u][t][4 * q + 1]), act(acc[u][t][4 * q + 2]), act(acc[u][t][4 * q + 3])};
            }
        flush(u0 * TILE, (uint32_t)0);
      }
    }
  };
  if (a.gelu == STT_GELU_NONE) leave([](float v) { return v; });
  else if (a.gelu == STT_GELU_TANH) leave([](float v) { return gelu1<STT_GELU_TANH>(v); });
  else leave([](float v) { return gelu1<STT_GELU_ERF>(v); });
}

unsigned grid_for(int64_t items) {
  const int64_t b = (items + 255) / 256;
  return (unsigned)(b < 1 ? 1 : b > 16384 ? 16384 : b);
}

// Tile and K split: MT from the rows; the widest NT that still gives kTileWaves waves (one a SIMD) with eight
// waves along K, so that activations are read as few times as possible; then the fewest waves along K that
// give as many, twice as many for a single row tile, whose blocks are short.  Measured, bf16 activations,
// us: 9 x 5 120 x 1 280: 3.4 (2 048 asked for: 4.0); 64 x 5 120 x 1 280: 5.7 (7.9); 150 x 1 280 x 5 120:
// 11.8 (20); one row x 51 866 x 1 280: 7.4 with two waves along K, 9.7 with one.
constexpr int64_t kTileWaves = 1024, kBigTiles = 144;
template <bool X4>
int launch_matmul(const stt_mxfp4_matmul_args& a, const Packed& p, bool vec, hipStream_t st) {
  const int64_t tiles_m = (a.m + 15) / 16;
  // Enough 128-row tiles for most compute units: the kernel that shares its operands through LDS.  160 tiles: 2 000 x
  // 1 280 x 5 120 bf16 51 us (56 in the other kernel), 1 000 x 5 120 x 1 280 in 4 bits 11.8 (16.4); 120 tiles: 300 x
  // 5 120 x 1 280 bf16 16.2 (14.1).  Few features leave most of a tile empty: 24 000 x 9 x 3 392 bf16 42 us (33).
  constexpr int BN = kBigFeatures<X4>;
  const bool vec16 = ((uintptr_t)a.d_out & 15) == 0 && a.out_row % (a.out_dtype == STT_F32 ? 4 : 8) == 0;
  const int64_t big_m = (a.m + 127) / 128, big_n = (a.n + BN - 1) / BN;
  const int64_t big_blocks = (big_m * big_n + 7) / 8 * 8;
  if (a.m >= 256 && a.n > 64 && a.k >= 128 && (X4 ? a.k : a.x_row) < 1 << 23 && big_m * big_n >= kBigTiles && big_blocks <= 0x7fffffff) {
    hipLaunchKernelGGL(mxfp4_matmul_big_kernel<X4>, dim3((unsigned)big_blocks), dim3(256), 0, st, a, (int)big_m, (int)big_n, vec16);
    return STT_OK;
  }
  int mt = tiles_m == 1 ? 1 : tiles_m == 2 || !X4 ? 2 : 4, nt = mt == 1 ? 2 : 4, wk = 1;
  const int64_t bm = (tiles_m + mt - 1) / mt;
  auto waves = [&](int t) { return bm * ((p.tiles_n + t - 1) / t); };
  while (nt > 1 && waves(nt) * 8 < kTileWaves) nt >>= 1;
  while (wk < 8 && waves(nt) * wk < (mt == 1 ? 2 * kTileWaves : kTileWaves) && wk * 2 <= p.chunks) wk <<= 1;
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
