// Quantisation to MXFP4, its inverse, and (Layer|RMS)Norm + adaLN modulation emitting MXFP4 (gfx950).
// The format and its formulas are in mxfp4_common.hpp.
//
// All three are bound by memory: 16-bit input is 2 bytes an element, the codes and scales 0.53. A block
// of 32 elements is four lanes of 8, so its maximum is a reduction inside a quad and nothing of a row has
// to wait for the rest of it (the per-token FP8 quantiser holds a whole row for one maximum).
#include "joy_common.hpp"
#include "joy_kernels.hpp"
#include "mxfp4_common.hpp"

namespace joy {
namespace {

template <int DT>  // 0 bf16, 1 fp16, 2 fp32
__device__ __forceinline__ float elem(const void* p, int64_t i) {
  if constexpr (DT == 0) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
  if constexpr (DT == 1) return fp16_bits_to_f32(((const uint16_t*)p)[i]);
  return ((const float*)p)[i];
}

// Eight consecutive elements as fp32; kVec: p + i is 16-byte aligned.
template <int DT, bool kVec>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&f)[8]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = elem<DT>(p, i + j);
  } else if constexpr (DT == 2) {
    const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    const uint4 v = *(const uint4*)((const uint16_t*)p + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = DT == 1 ? fp16_bits_to_f32(w[j] & 0xffffu) : bf16_lo(w[j]);
      f[2 * j + 1] = DT == 1 ? fp16_bits_to_f32(w[j] >> 16) : bf16_hi(w[j]);
    }
  }
}

// Where a lane's eight elements [k, k + 8) of a row go (k a multiple of 8, the quad holds one block): codes where
// k < K, the scale byte from the quad's first lane, where k lies in the last slab at least (past K: the unused bytes).
struct MxDest {
  uint8_t* q;
  uint8_t* s;
  __device__ __forceinline__ MxDest(uint8_t* codes, uint8_t* scales, int64_t row, int64_t k, int64_t K, int64_t slab_stride)
      : q(codes + row * (K >> 1) + (k >> 1)), s(scales + (k >> 8) * slab_stride + row * 8 + ((k >> 5) & 7)) {}
  __device__ __forceinline__ void store(uint32_t codes, uint32_t code, int64_t k, int64_t K) const {
    if ((k & 31) == 0 && k < ((K + kMxSlab - 1) & ~(int64_t)(kMxSlab - 1))) *s = (uint8_t)code;
    if (k < K) __builtin_nontemporal_store(codes, (uint32_t*)q);
  }
};

// Quantises eight values of the lane (zeros past K).
__device__ __forceinline__ void emit8(const float (&f)[8], const MxDest& d, int64_t k, int64_t K) {
  const uint32_t code = mx_code(quad_max_u32(abs_max8(f)));
  d.store(mx_pack8(f, mx_scale(code)), code, k, K);
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

// The same from eight packed 16-bit values: the maximum is taken of their bit patterns (they order like the
// magnitudes) and the conversion reads the 16-bit values themselves.
template <bool kFp16>
__device__ __forceinline__ void emit8_16bit(const u32x4& v, const MxDest& dst, int64_t k, int64_t K) {
  const uint32_t d[4] = {v[0], v[1], v[2], v[3]};  // (a bit cast of a vector's element itself takes element 0)
  us2 mx = __builtin_bit_cast(us2, d[0] & 0x7fff7fffu);
#pragma unroll
  for (int j = 1; j < 4; ++j) mx = __builtin_elementwise_max(mx, __builtin_bit_cast(us2, d[j] & 0x7fff7fffu));
  const uint32_t top = quad_max_u32(mx[0] > mx[1] ? mx[0] : mx[1]);
  const uint32_t code = mx_code(kFp16 ? __float_as_uint(fp16_bits_to_f32(top)) : top << 16);
  const float scale = mx_scale(code);
  uint32_t w = 0;
  if constexpr (kFp16) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2_vt, d[0]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2_vt, d[1]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2_vt, d[2]), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2_vt, d[3]), scale, 3);
  } else {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_vt, d[0]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_vt, d[1]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_vt, d[2]), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_vt, d[3]), scale, 3);
  }
  dst.store(w, code, k, K);
}

// One wave: 1024 consecutive elements of a row, 8 a lane in two strides, both loaded first.
template <int DT, bool kVec>
__global__ __launch_bounds__(256) void quant_mxfp4(MxQuantArgs a, int units_per_row) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = unit / units_per_row;
  if (row >= a.M) return;
  const int64_t k0 = (unit - row * units_per_row) * 1024 + (threadIdx.x & 63) * 8;
  auto dest = [&](int64_t k) { return MxDest(a.q, a.s, row, k, a.K, a.slab_stride); };
  if constexpr (kVec && DT != 2) {
    const uint16_t* x = (const uint16_t*)a.x + row * a.x_stride;
    u32x4 v[2] = {};
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (k0 + u * 512 < a.K) v[u] = __builtin_nontemporal_load((const u32x4*)(x + k0 + u * 512));
#pragma unroll
    for (int u = 0; u < 2; ++u) emit8_16bit<DT == 1>(v[u], dest(k0 + u * 512), k0 + u * 512, a.K);
  } else {
    float f[2][8] = {};
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (k0 + u * 512 < a.K) load8<DT, kVec>(a.x, row * a.x_stride + k0 + u * 512, f[u]);
#pragma unroll
    for (int u = 0; u < 2; ++u) emit8(f[u], dest(k0 + u * 512), k0 + u * 512, a.K);
  }
}

// One lane: 8 elements (a block's four lanes side by side), 4 times along the row.
template <int DT>
__global__ __launch_bounds__(256) void dequant_mxfp4(const uint8_t* __restrict__ q, const uint8_t* __restrict__ s,
                                                     int64_t slab_stride, void* __restrict__ out, int64_t M, int64_t K,
                                                     int units_per_row) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = unit / units_per_row;
  if (row >= M) return;
  const int64_t k0 = (unit - row * units_per_row) * 2048 + (threadIdx.x & 63) * 8;
  uint32_t w[4], code[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t k = k0 + u * 512;
    if (k >= K) continue;
    w[u] = __builtin_nontemporal_load((const uint32_t*)(q + row * (K >> 1) + (k >> 1)));
    code[u] = s[(k >> 8) * slab_stride + row * 8 + ((k >> 5) & 7)];
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t k = k0 + u * 512;
    if (k >= K) continue;
    const float scale = mx_scale(code[u]);
    const bool nan = code[u] == 255;  // whatever the elements
    if constexpr (DT == 0) {
      // bf16 holds every product of an element and a scale below 2^127 (exact)
      const uint32_t p[4] = {
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[u], scale, 0)),
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[u], scale, 1)),
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[u], scale, 2)),
          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[u], scale, 3))};
      const u32x4 v = {nan ? 0x7fc07fc0u : p[0], nan ? 0x7fc07fc0u : p[1], nan ? 0x7fc07fc0u : p[2], nan ? 0x7fc07fc0u : p[3]};
      __builtin_nontemporal_store(v, (u32x4*)((uint16_t*)out + row * K + k));
    } else {
      const f32x2_vt c[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], scale, 0),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], scale, 1),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], scale, 2),
                             __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], scale, 3)};
      uint32_t p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = nan ? 0x7fc00000u : __float_as_uint(c[j >> 1][j & 1]);
      if constexpr (DT == 2) {
        u32x4* o = (u32x4*)((float*)out + row * K + k);
        __builtin_nontemporal_store((u32x4){p[0], p[1], p[2], p[3]}, o);
        __builtin_nontemporal_store((u32x4){p[4], p[5], p[6], p[7]}, o + 1);
      } else {
        u32x4 h;
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = pack_fp16x2(__uint_as_float(p[2 * j]), __uint_as_float(p[2 * j + 1]));
        __builtin_nontemporal_store(h, (u32x4*)((uint16_t*)out + row * K + k));
      }
    }
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// Sum over the wave in its last lane, in the DPP network (no LDS crossbar).
template <int kCtrl, int kRows>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, kRows, 0xf, false));
}
__device__ __forceinline__ float wave_sum_last(float v) {
  v = dpp_add<0xB1, 0xf>(v);     // quad_perm [1, 0, 3, 2]
  v = dpp_add<0x4E, 0xf>(v);     // quad_perm [2, 3, 0, 1]
  v = dpp_add<0x141, 0xf>(v);    // row_half_mirror: eight lanes
  v = dpp_add<0x140, 0xf>(v);    // row_mirror: sixteen
  v = dpp_add<0x142, 0xa>(v);    // row_bcast15 into rows 1 and 3
  return dpp_add<0x143, 0xc>(v); // row_bcast31 into rows 2 and 3
}

// Eight values as loaded, converted only when they are used. Loads past the range give zeros.
template <int DT>
struct Raw8 {
  u32x4 v[DT == 2 ? 2 : 1];
  template <int kAux>
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int lane_at, int at) {  // in values
    constexpr int ESZ = DT == 2 ? 4 : 2;
    v[0] = __builtin_amdgcn_raw_buffer_load_b128(r, lane_at * ESZ, at * ESZ, kAux);
    if constexpr (DT == 2) v[1] = __builtin_amdgcn_raw_buffer_load_b128(r, lane_at * ESZ + 16, at * ESZ, kAux);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == 2) {
        f[j] = __uint_as_float(v[0][j]);
        f[4 + j] = __uint_as_float(v[1][j]);
      } else {
        const uint32_t w = v[0][j];
        f[2 * j] = DT == 1 ? fp16_bits_to_f32(w & 0xffffu) : bf16_lo(w);
        f[2 * j + 1] = DT == 1 ? fp16_bits_to_f32(w >> 16) : bf16_hi(w);
      }
    }
  }
};

// One row per workgroup of N / 8 / VPT threads, rounded up to waves: VPT vectors of 8 values a lane, all loaded at once.
// Of 3120 x 5120's 11.8 us the bytes are 8.0 at a large copy's rate and the vector instructions 6.3, 248 a lane for 16
// elements; the rest is where a row waits for its two sums in turn. So nothing in it branches: lanes behind the row
// load zeros, have no part in the sums and store nothing, by their buffers' ranges (with branches, sums over the LDS
// crossbar and two-operand maxima, 365: 3120 x 5120 15.1 us against 11.8, 10800 x 5120 42 against 31.5, 4.4 TB/s). A
// wave per row leaves too few loads in flight (3120 x 4096 16.8 against 9.4 us); workgroups that walk the rows with the
// next one's loads ahead and the modulation in registers hold fewer waves (10800 x 5120 4 us slower than without).
constexpr int kRowWaves = 8;  // at most
constexpr int kNt = 2;        // a buffer access's nontemporal bit

template <int DT, int NORM, int VPT, bool kAffine>
__global__ __launch_bounds__(64 * kRowWaves) void norm_mod_mxfp4_rows(NormModArgs a, int64_t slab_stride, float inv_n) {
  __shared__ __attribute__((aligned(16))) float red[2][kRowWaves];
  constexpr int ESZ = DT == 2 ? 4 : 2;
  const int T = blockDim.x, t = threadIdx.x, N = (int)a.N;
  const int64_t row = blockIdx.x, mb = a.mod_rows == 1 ? 0 : row;
  auto range = [](const void* p, int bytes) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00020000); };
  auto row_of = [&](const void* p, int64_t first) { return range((const char*)p + first * ESZ, N * ESZ); };
  const auto xr = row_of(a.x, row * a.x_stride), scr = row_of(a.scale, mb * a.N), shr = row_of(a.shift, mb * a.N);
  Raw8<DT> raw[VPT], sc[VPT], sh[VPT], ga[kAffine ? VPT : 1], be[kAffine && NORM == 0 ? VPT : 1];
#pragma unroll
  for (int i = 0; i < VPT; ++i) raw[i].template load<kNt>(xr, t * 8, i * T * 8);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    sc[i].template load<0>(scr, t * 8, i * T * 8);
    sh[i].template load<0>(shr, t * 8, i * T * 8);
  }
  if constexpr (kAffine) {
    const auto gr = row_of(a.gamma, 0);
#pragma unroll
    for (int i = 0; i < VPT; ++i) ga[i].template load<0>(gr, t * 8, i * T * 8);
    if constexpr (NORM == 0) {
      // without beta an empty range at scalar offset 0: zeros
      const auto br = range(a.beta, a.beta ? N * ESZ : 0);
      const int step = a.beta ? T * 8 : 0;
#pragma unroll
      for (int i = 0; i < VPT; ++i) be[i].template load<0>(br, t * 8, i * step);
    }
  }
  if (t < 2 * kRowWaves && (t & (kRowWaves - 1)) >= T >> 6) (&red[0][0])[t] = 0.f;  // waves that the workgroup lacks
  auto row_mean = [&](float v, int slot) {
    v = wave_sum_last(v);
    if ((t & 63) == 63) red[slot][t >> 6] = v;
    __syncthreads();
    const float4 p = *(const float4*)&red[slot][0], q = *(const float4*)&red[slot][4];
    return (((p.x + p.y) + (p.z + p.w)) + ((q.x + q.y) + (q.z + q.w))) * inv_n;
  };
  float x[VPT][8], sum = 0.f, mean = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) raw[i].get(x[i]);
  if constexpr (NORM == 0) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += x[i][j];
    mean = row_mean(sum, 0);
    sum = 0.f;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const float m = (t + i * T) * 8 < N ? mean : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[i][j] -= m;
      sum = __builtin_fmaf(x[i][j], x[i][j], sum);
    }
  }
  const float rstd = __builtin_amdgcn_rsqf(row_mean(sum, 1) + a.eps);
  const int nslabs = (N + kMxSlab - 1) / kMxSlab;
  const auto qr = range((uint8_t*)a.out_q + row * (N >> 1), N >> 1);
  const auto sr = range((uint8_t*)a.out_s + row * 8, (int)((nslabs - 1) * slab_stride) + 8);
  // the quad's first lane stores its scale, also the unused bytes of the last slab
  const uint32_t slab = (uint32_t)slab_stride, s_at = (t & 3) == 0 ? (t >> 5) * slab + ((t >> 2) & 7) : 0x7fffffffu;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const float r = (t + i * T) * 8 < N ? rstd : 0.f;
    float y[8], m[8], add[8];
    sc[i].get(m);
    sh[i].get(add);
    if constexpr (kAffine) {
      float g[8], b[8] = {};
      ga[i].get(g);
      if constexpr (NORM == 0) be[i].get(b);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = __builtin_fmaf(__builtin_fmaf(x[i][j] * r, g[j], b[j]), 1.f + m[j], add[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = __builtin_fmaf(x[i][j] * r, 1.f + m[j], add[j]);
    }
    const uint32_t code = mx_code(quad_max_u32(abs_max8(y)));
    __builtin_amdgcn_raw_buffer_store_b32(mx_pack8(y, mx_scale(code)), qr, t * 4, i * T * 4, kNt);
    __builtin_amdgcn_raw_buffer_store_b8((uint8_t)code, sr, (int)s_at, (int)(i * (T >> 5) * slab), 0);
  }
}

// One wave per row, any length and alignment: the row is read once for each of mean, variance and result
// (cached after the first), and the modulated values are quantised as they are, in fp32.
template <int DT, int NORM, bool kVec>
__global__ __launch_bounds__(256) void norm_mod_mxfp4(NormModArgs a, int64_t slab_stride) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.M) return;
  const int64_t xb = row * a.x_stride, mb = (a.mod_rows == 1 ? 0 : row) * a.N;
  float sum = 0.f, mean = 0.f;
  for (int64_t k = lane * 8; k < a.N; k += 512) {
    float f[8];
    load8<DT, kVec>(a.x, xb + k, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += NORM == 0 ? f[j] : f[j] * f[j];
  }
  if constexpr (NORM == 0) {
    mean = wave_sum(sum) / (float)a.N;
    sum = 0.f;
    for (int64_t k = lane * 8; k < a.N; k += 512) {
      float f[8];
      load8<DT, kVec>(a.x, xb + k, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += (f[j] - mean) * (f[j] - mean);
    }
  }
  const float r = __builtin_amdgcn_rsqf(wave_sum(sum) / (float)a.N + a.eps);
  for (int64_t k0 = 0; k0 < a.N; k0 += 512) {  // whole quads: the block's maximum is a quad reduction
    const int64_t k = k0 + lane * 8;
    float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k < a.N) {
      float f[8], sc[8], sh[8], g[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, b[8] = {};
      load8<DT, kVec>(a.x, xb + k, f);
      load8<DT, kVec>(a.scale, mb + k, sc);
      load8<DT, kVec>(a.shift, mb + k, sh);
      if (a.gamma) load8<DT, kVec>(a.gamma, k, g);
      if (a.beta && NORM == 0) load8<DT, kVec>(a.beta, k, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float n = NORM == 0 ? (f[j] - mean) * r * g[j] + b[j] : f[j] * r * g[j];
        y[j] = n * (1.f + sc[j]) + sh[j];
      }
    }
    emit8(y, MxDest((uint8_t*)a.out_q, (uint8_t*)a.out_s, row, k, a.N, slab_stride), k, a.N);
  }
}

template <int DT>
hipError_t launch_quant(const MxQuantArgs& a, hipStream_t st) {
  const int upr = (int)((a.K + 1023) / 1024);
  const dim3 grid((unsigned)((a.M * upr + 3) / 4));
  const int esz = DT == 2 ? 4 : 2;
  // rows that are not 16-byte aligned are read element by element (10800 x 13824 75.7 us against 67.3)
  if ((uintptr_t)a.x % 16 == 0 && a.x_stride * esz % 16 == 0)
    hipLaunchKernelGGL((quant_mxfp4<DT, true>), grid, dim3(256), 0, st, a, upr);
  else
    hipLaunchKernelGGL((quant_mxfp4<DT, false>), grid, dim3(256), 0, st, a, upr);
  return hipGetLastError();
}

template <int DT, int NORM>
hipError_t launch_norm(const NormModArgs& a, int64_t slab_stride, hipStream_t st) {
  const int esz = DT == 2 ? 4 : 2;
  const bool vec = (uintptr_t)a.x % 16 == 0 && a.x_stride * esz % 16 == 0 && (uintptr_t)a.scale % 16 == 0 &&
                   (uintptr_t)a.shift % 16 == 0 && (uintptr_t)a.gamma % 16 == 0 && (uintptr_t)a.beta % 16 == 0;
  // Rows that are not 16-byte aligned (3120 x 4096 17.9 us against 8.6) and those of more than four vectors a lane (1560
  // x 16416 48, where 1560 x 16384 takes 16) go to the general kernel. One vector a lane, not two, past 256 of them:
  // 3120 x 4096 10.8 us against 9.4; four, not two, past 512: level.
  if (vec && a.N <= 16384) {
    // whole slabs of vectors between a lane's, so that its destinations lie at one distance
    const int nvec = (int)(a.N / 8), vpt = nvec <= 256 ? 1 : nvec <= 1024 ? 2 : 4;
    const int threads = ((nvec + vpt - 1) / vpt + 63) / 64 * 64;
    auto kern = a.gamma ? (vpt == 1   ? norm_mod_mxfp4_rows<DT, NORM, 1, true>
                           : vpt == 2 ? norm_mod_mxfp4_rows<DT, NORM, 2, true>
                                      : norm_mod_mxfp4_rows<DT, NORM, 4, true>)
                        : (vpt == 1   ? norm_mod_mxfp4_rows<DT, NORM, 1, false>
                           : vpt == 2 ? norm_mod_mxfp4_rows<DT, NORM, 2, false>
                                      : norm_mod_mxfp4_rows<DT, NORM, 4, false>);
    hipLaunchKernelGGL(kern, dim3((unsigned)a.M), dim3(threads), 0, st, a, slab_stride, 1.f / (float)a.N);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)((a.M + 3) / 4));
  if (vec)
    hipLaunchKernelGGL((norm_mod_mxfp4<DT, NORM, true>), grid, dim3(256), 0, st, a, slab_stride);
  else
    hipLaunchKernelGGL((norm_mod_mxfp4<DT, NORM, false>), grid, dim3(256), 0, st, a, slab_stride);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_quant_mxfp4(const MxQuantArgs& a, hipStream_t st) {
  if (a.dtype == 0) return launch_quant<0>(a, st);
  return a.dtype == 1 ? launch_quant<1>(a, st) : launch_quant<2>(a, st);
}

hipError_t launch_dequant_mxfp4(const void* q, const void* s, int64_t slab_stride, void* out, int dtype, int64_t M,
                                int64_t K, hipStream_t st) {
  const int upr = (int)((K + 2047) / 2048);
  auto kern = dtype == 0 ? dequant_mxfp4<0> : dtype == 1 ? dequant_mxfp4<1> : dequant_mxfp4<2>;
  hipLaunchKernelGGL(kern, dim3((unsigned)((M * upr + 3) / 4)), dim3(256), 0, st, (const uint8_t*)q, (const uint8_t*)s,
                     slab_stride, out, M, K, upr);
  return hipGetLastError();
}

hipError_t launch_norm_modulate_mxfp4(const NormModArgs& a, int64_t slab_stride, hipStream_t st) {
  if (a.norm_type == 0) {
    if (a.dtype == 0) return launch_norm<0, 0>(a, slab_stride, st);
    return a.dtype == 1 ? launch_norm<1, 0>(a, slab_stride, st) : launch_norm<2, 0>(a, slab_stride, st);
  }
  if (a.dtype == 0) return launch_norm<0, 1>(a, slab_stride, st);
  return a.dtype == 1 ? launch_norm<1, 1>(a, slab_stride, st) : launch_norm<2, 1>(a, slab_stride, st);
}

}  // namespace joy
