// MXFP4 x MXFP4 -> bf16 / fp16 GEMM with block scales and fused epilogue, gfx950.
//
//   acc[m, n] = sum_k A[m, k] W[n, k]      A, W: E2M1 elements times their blocks' E8M0 scales, the
//                                          products exact and summed in fp32 by the MFMA
//   y = acc + bias[n]
//   out = round(y)                                     plain
//   out = round(gelu_tanh(y))                          GELU
//   out = round(residual[m, n] + y * gate[n])          gated residual (in place where out == residual)
//   out = MXFP4(gelu_tanh(y))                          GELU, quantised for the next product
//
// Everything up to the one rounding at the end is fp32: a rounding to 16 bits before the GELU, the gate or
// the quantiser would add half a step of that type to each value (before the quantiser it moves one
// element in some hundred to the neighbouring code).
//
// v_mfma_scale_f32_32x32x64_f8f6f4 applies the scales itself: lane l holds 32 consecutive elements (16
// bytes, one block) of row l % 32 and, in one byte of a register, their scale. W is the instruction's
// first operand, so that a lane ends up with one row m = l % 32 and, in groups of four, the columns
// n = 8 (r / 4) + 4 (l / 32) + r % 4 of accumulator r: the 32 columns of a tile are an MXFP4 block of the
// row, shared by lanes l and l ^ 32.
#include <algorithm>
#include <type_traits>

#include "gemm_common.hpp"
#include "joy_common.hpp"
#include "joy_kernels.hpp"
#include "mxfp4_common.hpp"
#include "mxfp4_schedule.hpp"

namespace joy {
namespace {

constexpr int kGroup = 4;  // tile rows that walk the tile columns together

enum Epi : int { kPlain = 0, kGelu = 1, kResidual = 2, kGeluQuant = 3 };

// Byte kByte of the scale registers is the one that counts.
template <int kByte>
__device__ __forceinline__ v16f mfma_fp4(const v4i& a, const v4i& b, const v16f& c, int sa, int sb) {
  const v8i a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, kByte, sa, kByte, sb);
}

template <bool kBf16>
__device__ __forceinline__ float value16(uint32_t bits) {
  if constexpr (kBf16) return __uint_as_float(bits << 16);
  return fp16_bits_to_f32(bits);
}

__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xc07f); }

template <int J>
using IC = std::integral_constant<int, J>;

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <bool kBf16>
__device__ __forceinline__ uint32_t pack16x2(float lo, float hi) {
  if constexpr (kBf16) return pack_bf16x2(lo, hi);
  return pack_fp16x2(lo, hi);
}
template <bool kBf16>
__device__ __forceinline__ float lo16(uint32_t w) {
  return value16<kBf16>(w & 0xffffu);
}
template <bool kBf16>
__device__ __forceinline__ float hi16(uint32_t w) {
  return value16<kBf16>(w >> 16);
}

// kN MFMAs, a group of LDS reads after each of the first ones until kReads are placed.
template <int I, int kN, int kReads>
__device__ __forceinline__ void interleave_reads() {
  if constexpr (I < kN) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    constexpr int kPer = (kReads + kN - 1) / kN;
    if constexpr (I * kPer < kReads) __builtin_amdgcn_sched_group_barrier(0x100, kPer, 0);
    interleave_reads<I + 1, kN, kReads>();
  }
}

// Persistent kernel: gridDim.x workgroups walk the tiles b, b + gridDim.x, ... of the XCD-ordered grouped tile
// order. Tile BM x BN = 64 FM x 64 FN, four waves in 2 x 2, each FM x FN MFMA tiles of 32 x 32.
//
// K runs in slabs of 256 elements (128 bytes a row, one slab of scales) through an LDS ring of S slabs (two at
// 256 x 256, up to four of smaller tiles) that goes on across tiles. Lane l takes chunks (16 bytes, one block) 4 (l / 32) + t of row l % 32 in MFMA step t = 0..3, for both
// operands, so that its four scales are one aligned dword of the row's eight scale bytes and t selects the byte. Chunk
// c of row r is stored at c ^ swz(r), swz(r) = (r & 7) ^ ((r >> 3) & 1): sixteen lanes of consecutive rows read
// sixteen different 16-byte columns of 256 bytes.
//
// All of a slab's fragments are in registers by the middle of its MFMAs. The first phase takes W units [0, FN / 2)
// against every A unit, A unit after A unit, and reads the other W units; the second takes those and reads the next
// slab's first W units, its scales and, unit after unit, its A fragments into the registers that the MFMAs leave. So a
// slab's A rows in LDS are free when its MFMAs begin and its W rows in their middle: the loads of the A rows S slabs
// ahead go out in the first phase, those of the W rows and scales in the second, each behind a barrier, and have S -
// 1 / 2 and S - 1 slabs to land. With both issued together, one slab ahead, the MFMAs of 10800 x 5120 x 15360
// waited 0.9 of every 1.9 us a slab; in half slabs of 64 bytes a row, three ahead, as long: L2 gives 64-byte rows
// half the rate (14 against 25 TB/s).
//
// Rows past M or N fall outside the buffer descriptors and load zeros; so do the elements past K of the last row,
// while other rows' elements past K are whatever follows them, under scale bytes that are 0 in both operands: 2^-254
// times at most 36 is 0 in fp32.
//
// What bounds it: with many tiles a CU the power. 10800 x 5120 x 15360 takes 376 us (4.52 PFLOP/s) at 1.69 GHz with the
// MFMAs 63 % busy, 297 us with zeros for data (a loop of these MFMAs on registers alone reaches 6.7). In one round of
// tiles operands arrive at 35 (from HBM) to 45 (from the last-level cache) bytes a ns and CU, half of what L2 gives 128-
// byte rows; why no faster has not been found. The 256 x 256 kernels spill 56 to 72 bytes: in a tile's first slab a
// reloaded address waits for every load and store in flight, and addresses reloaded behind the epilogue's stores wait
// for these, so that each tile drains the ring's loads once or twice. The smaller tiles have no scratch.
//
// A workgroup's tiles of one shape: run_tiles() for main tiles, then for the rest's smaller ones (MxTilePlan).
struct MxTilePlan {
  int tiles_m, tiles_n;  // grid of main tiles
  int main;              // tiles_m * tiles_n
  int rest;              // rest tiles: the rows past those of the grid, tile row after tile row
  int rest_wgs;          // workgroups that take them
};

// Tile `b` of a launch: its first row and column.
struct MxOrigin {
  int64_t m0;
  int n0;
};
template <int BM, int BN, int kMainRows, bool kRest>
__device__ __forceinline__ MxOrigin tile_origin(const MxTilePlan& p, int b) {
  if constexpr (!kRest) {
    const TileCoord tc = map_tile(b, p.main, p.tiles_m, p.tiles_n, kGroup, 0);
    return {(int64_t)tc.tm * BM, tc.tn * BN};
  } else {
    return {(int64_t)p.tiles_m * kMainRows + (int64_t)(b / p.tiles_n) * BM, b % p.tiles_n * BN};
  }
}

constexpr int tiles_lds(int FM, int FN) {  // of one slab: operand rows and scales
  return 64 * (FM + FN) * 128 + ((64 * FM + 127) / 128 + (64 * FN + 127) / 128) * 1024;
}
constexpr int kStagePitch = 144, kStageBytes = 32 * kStagePitch;  // a wave's staged rows of 128 bytes in the epilogue

// Tiles first, first + P, ... below count.
template <bool kBf16, int kEpi, int FM, int FN, int S, int kMainRows, bool kRest>
__device__ __forceinline__ void run_tiles(const MxGemmArgs& g, const MxTilePlan& plan, int first, int P, int count,
                                          uint8_t* lds, uint8_t* side, uint8_t* stage_lds) {
  constexpr int BM = 64 * FM, BN = 64 * FN, RB = 128;
  constexpr int IA = BM / 32, IW = BN / 32;                    // 1 KB loads a wave and slab
  constexpr int NA = (BM + 127) / 128, NW = (BN + 127) / 128;  // 1 KB scale loads a workgroup and slab
  constexpr int W_OFF = BM * RB, SA_OFF = W_OFF + BN * RB, SW_OFF = SA_OFF + NA * 1024;
  constexpr int SLAB = SW_OFF + NW * 1024;
  constexpr MxTileCounts kCounts = {FM, FN, S, kEpi == kGeluQuant};
  constexpr int PITCH = kStagePitch;
  constexpr int FA = FN / 2;  // W units of a slab's first phase
  static_assert(IA == kCounts.a() && IW == kCounts.w(), "loads of a slab");
  static_assert(SLAB == tiles_lds(FM, FN) && S >= 2 && kCounts.next_slab_first() < 64, "LDS, vmcnt range");

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int Kb = g.K >> 1, nk = (g.K + 255) >> 8;
  const uint32_t lds0 = lds_u32((lds_void*)lds), side0 = lds_u32((lds_void*)side);
  // absent bias: an empty range, which loads zeros
  const __amdgpu_buffer_rsrc_t brs =
      __builtin_amdgcn_make_buffer_rsrc((void*)g.bias, 0, g.bias ? g.N * 2 : 0, 0x00020000);
  const __amdgpu_buffer_rsrc_t grs =
      __builtin_amdgcn_make_buffer_rsrc((void*)g.gate, 0, kEpi == kResidual ? g.N * 2 : 0, 0x00020000);
  if (first >= count) return;

  // ---- the stream of loads
  __amdgpu_buffer_rsrc_t ars, wrs, srs;
  uint32_t oa[IA], ow[IW], os = 0;
  const int sidx = wave % (NA + NW);  // this wave's scale load (waves past the last repeat one: the same bytes)
  const bool s_is_a = sidx < NA;
  const uint32_t s_lds = s_is_a ? SA_OFF + sidx * 1024 : SW_OFF + (sidx - NA) * 1024;
  const int s_step = (int)(s_is_a ? g.slab_a : g.slab_b);
  MxLoadStream at = {first, RB, s_step};
  auto load_tile = [&](int b) {
    const MxOrigin o = tile_origin<BM, BN, kMainRows, kRest>(plan, b);
    const int64_t m0 = o.m0;
    const int n0 = mx_load_column(o.n0, g.N);
    const int rows = (int)min((int64_t)BM, g.M - m0), cols = min(BN, g.N - n0);
    ars = __builtin_amdgcn_make_buffer_rsrc((uint8_t*)g.A + m0 * Kb, 0, rows * Kb, 0x00020000);
    wrs = __builtin_amdgcn_make_buffer_rsrc((uint8_t*)g.W + (int64_t)n0 * Kb, 0, cols * Kb, 0x00020000);
    const uint8_t* sp = s_is_a ? (const uint8_t*)g.scales_a + m0 * 8 : (const uint8_t*)g.scales_b + (int64_t)n0 * 8;
    const int64_t end = (int64_t)(nk - 1) * s_step + (s_is_a ? g.M - m0 : g.N - n0) * 8;
    srs = __builtin_amdgcn_make_buffer_rsrc((uint8_t*)sp, 0, (int)end, 0x00020000);
    const int lrow = lane >> 3, lchunk = lane & 7;  // 8 rows a load
#pragma unroll
    for (int i = 0; i < IA; ++i) {
      const int row = (wave * IA + i) * 8 + lrow;
      oa[i] = (uint32_t)row * (uint32_t)Kb + (uint32_t)((lchunk ^ (row & 7) ^ ((row >> 3) & 1)) * 16);
    }
#pragma unroll
    for (int i = 0; i < IW; ++i) {
      const int row = (wave * IW + i) * 8 + lrow;
      ow[i] = (uint32_t)row * (uint32_t)Kb + (uint32_t)((lchunk ^ (row & 7) ^ ((row >> 3) & 1)) * 16);
    }
    os = (uint32_t)((s_is_a ? sidx : sidx - NA) * 1024 + lane * 16);
  };
  // load number d of the slab's A rows, and of its W rows and (the last) scales
  // (the range check of a raw buffer includes the scalar offset)
  auto load_a = [&](int d, uint32_t slab) { dma_buf16(slab + (wave * IA + d) * 1024, oa[d], ars, at.k_off); };
  auto load_w = [&](int d, uint32_t slab) {
    if (d < IW)
      dma_buf16(slab + W_OFF + (wave * IW + d) * 1024, ow[d], wrs, at.k_off);
    else
      dma_buf16(slab + s_lds, os, srs, at.s_off);
  };
  // before a slab's loads: on to the next tile after the last slab of one, and to loads that fetch nothing after the
  // last tile. Outside the slab's code, whose MFMAs stay in place only in one basic block
  auto aim = [&]() {
    if (at.next(nk, P, count, RB, s_step)) {
      if (at.tile < count) {
        load_tile(at.tile);
      } else {
        ars = wrs = srs = __builtin_amdgcn_make_buffer_rsrc((uint8_t*)g.A, 0, 0, 0x00020000);
      }
    }
  };

  // bias (odd waves, with a residual: gate) of the columns from n0 on; side_at: the half of `side` that holds this tile's
  uint32_t side_at = 0;
  auto load_side = [&](int n0, uint32_t at) {
    const bool gate = kEpi == kResidual && (wave & 1);
    dma_buf16(side0 + at + (gate ? 1024 : 0), (uint32_t)(n0 + lane * 8) * 2, gate ? grs : brs, 0);
  };

  // ---- fragments
  const int frow = lane & 31, half = lane >> 5, fsw = (frow & 7) ^ ((frow >> 3) & 1);
  uint32_t fo[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) fo[t] = (uint32_t)(((4 * half + t) ^ fsw) * 16 + frow * RB);
  const uint32_t a_wave = wm * (BM / 2) * RB, w_wave = W_OFF + wn * (BN / 2) * RB;
  const uint32_t sa_wave = SA_OFF + (wm * (BM / 2) + frow) * 8 + half * 4;
  const uint32_t sw_wave = SW_OFF + (wn * (BN / 2) + frow) * 8 + half * 4;
  v16f acc[FN][FM];
  v4i fa[FM][4], fw[FN][4];
  int sa[FM], sw[FN], sa_next[FM], sw_next[FN];
  auto read_a1 = [&](int j, int t, uint32_t slab) {
    fa[j][t] = *(const v4i*)(lds + slab + a_wave + fo[t] + j * 32 * RB);
  };
  auto read_a = [&](int j, uint32_t slab) {
#pragma unroll
    for (int t = 0; t < 4; ++t) read_a1(j, t, slab);
  };
  auto read_w = [&](int i, uint32_t slab) {
#pragma unroll
    for (int t = 0; t < 4; ++t) fw[i][t] = *(const v4i*)(lds + slab + w_wave + fo[t] + i * 32 * RB);
  };
  auto read_scales = [&](uint32_t slab) {
#pragma unroll
    for (int j = 0; j < FM; ++j) sa_next[j] = *(const int*)(lds + slab + sa_wave + j * 256);
#pragma unroll
    for (int i = 0; i < FN; ++i) sw_next[i] = *(const int*)(lds + slab + sw_wave + i * 256);
  };
  auto mma = [&](auto tc, auto zero, int i, int j) {
    constexpr int t = decltype(tc)::value;
    acc[i][j] = mfma_fp4<t>(fw[i][t], fa[j][t], decltype(zero)::value && t == 0 ? (v16f){} : acc[i][j], sw[i], sa[j]);
  };
  uint32_t slab = 0;
  // one slab; wait: loads and stores that may still be in flight when the last phase begins
  auto slab_step = [&](auto zero, auto wait, int n_next) {
    constexpr bool kFirst = decltype(zero)::value;
#pragma unroll
    for (int j = 0; j < FM; ++j) sa[j] = sa_next[j];
#pragma unroll
    for (int i = 0; i < FN; ++i) sw[i] = sw_next[i];
    const uint32_t next = slab == (S - 1) * SLAB ? 0 : slab + SLAB, dst = lds0 + slab;
    // the MFMAs of W units [i0, i1) against A unit j; after(n) follows the n-th of them
    auto unit = [&](int i0, int i1, int j, auto after) {
      int n = 0;
      auto row = [&](auto tc) {
#pragma unroll
        for (int i = i0; i < i1; ++i) {
          mma(tc, zero, i, j);
          after(n++);
        }
      };
      row(IC<0>{}), row(IC<1>{}), row(IC<2>{}), row(IC<3>{});
    };
    // first phase: W units [0, FA), while the others are read
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = FA; i < FN; ++i) read_w(i, slab);
    unit(0, FA, 0, [](int) {});
    interleave_reads<0, 4 * FA, 4 * (FN - FA)>();
    __builtin_amdgcn_sched_barrier(0);
    // every wave has read this slab's A rows, the last of them a unit ago: in their place come those of S slabs on
    wait_lgkm0();
    block_barrier();
    __builtin_amdgcn_sched_barrier(0);
    constexpr int kLeft = 4 * FA * (FM - 1);  // MFMAs of this phase that are left
    if constexpr (kLeft == 0) {
#pragma unroll
      for (int d = 0; d < IA; ++d) load_a(d, dst);
    }
#pragma unroll
    for (int j = 1; j < FM; ++j)
      unit(0, FA, j, [&](int n) {
        const int at = 4 * FA * (j - 1) + n;
#pragma unroll
        for (int d = at * IA / (kLeft + !kLeft); d < (at + 1) * IA / (kLeft + !kLeft); ++d) load_a(d, dst);
        __builtin_amdgcn_sched_barrier(0);
      });
    wait_vmcnt_lgkm0<decltype(wait)::value>();
    block_barrier();
    __builtin_amdgcn_sched_barrier(0);
    // second phase: the next slab has landed for every wave, this slab's W rows have been read and the last tile's
    // epilogue is over
    if constexpr (kFirst) load_side(n_next, 2048 - side_at);
    constexpr int kN = 4 * (FN - FA);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      unit(FA, FN, j, [&](int n) {
        const int at = kN * j + n;
        if (at < FA) read_w(at, next);
        if (at == FA) read_scales(next);
        if (j > 0 && n % (kN / 4) == kN / 4 - 1) read_a1(j - 1, n / (kN / 4), next);
#pragma unroll
        for (int d = at * (IW + 1) / (kN * FM); d < (at + 1) * (IW + 1) / (kN * FM); ++d) load_w(d, dst);
        __builtin_amdgcn_sched_barrier(0);
      });
    }
    read_a(FM - 1, next);
    // the accumulators stay where they are across blocks (no instruction)
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) asm volatile("" : "+a"(acc[i][j]));
    slab = next;
  };

  // ---- epilogue of a tile. Unit (i, j) is 32 columns x 32 rows; a swap of two accumulator quads between lanes l and
  // l ^ 32 gives each lane eight consecutive columns, 16 p + 8 half, of row l % 32, for p = 0 and 1. Results pass
  // through the wave's staging rows so that a store covers 128 (residual and MXFP4: 64) bytes of a row: 32-byte
  // pieces straight from the lanes made four times the requests.
  auto epilogue = [&](int64_t m0, int n0) {
    int le;  // an opaque copy of the lane index keeps the addresses below out of the main loop's registers
    asm volatile("v_mov_b32 %0, %1" : "=v"(le) : "v"(lane));
    const int er = le & 31, eh = le >> 5;
    uint8_t* stage = stage_lds + wave * kStageBytes;
    const int rows = (int)min((int64_t)BM, g.M - m0);
    const int r0 = wm * (BM / 2), c0 = n0 + wn * (BN / 2);  // the wave's first row of the tile and its first column
    auto columns = [&](int i, int j, int p, float (&y)[8]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[i][j][8 * p + e]),
                                                        __float_as_uint(acc[i][j][8 * p + 4 + e]), false, false);
        y[e] = __uint_as_float(r[0]);
        y[4 + e] = __uint_as_float(r[1]);
      }
    };
    // eight values of the tile's bias or gate from the wave's column c
    auto side8 = [&](int at, int c, float (&v)[8]) {
      const uint4 w = *(const uint4*)(side + side_at + at + (wn * (BN / 2) + c) * 2);
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = lo16<kBf16>(x[e]);
        v[2 * e + 1] = hi16<kBf16>(x[e]);
      }
    };
    if constexpr (kEpi == kGeluQuant) {
      const int nslabs = (g.N + 255) >> 8;
      const __amdgpu_buffer_rsrc_t crs = __builtin_amdgcn_make_buffer_rsrc(
          (uint8_t*)g.C + m0 * (g.N >> 1), 0, rows * (g.N >> 1), 0x00020000);
      const __amdgpu_buffer_rsrc_t scr = __builtin_amdgcn_make_buffer_rsrc(
          (uint8_t*)g.out_s + m0 * 8, 0, (int)((nslabs - 1) * g.slab_c + rows * 8), 0x00020000);
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        uint32_t codes = 0;
#pragma unroll
        for (int i = 0; i < FN; ++i) {
          float y[2][8];
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            float b[8];
            side8(0, i * 32 + 16 * p + 8 * eh, b);
            columns(i, j, p, y[p]);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[p][e] = gelu_tanh(y[p][e] + b[e]);
          }
          const uint32_t top[2] = {abs_max8(y[0]), abs_max8(y[1])}, mx = top[0] > top[1] ? top[0] : top[1];
          const auto r = __builtin_amdgcn_permlane32_swap(mx, mx, false, false);
          const uint32_t code = mx_code(r[0] > r[1] ? r[0] : r[1]);
          codes |= (c0 + i * 32 < g.N ? code : 0) << (8 * i);
#pragma unroll
          for (int p = 0; p < 2; ++p)  // bytes 16 i + 8 p + 4 half of the wave's part of the row
            *(uint32_t*)(stage + er * 80 + i * 16 + p * 8 + eh * 4) = mx_pack8(y[p], mx_scale(code));
        }
        constexpr int CPL = FN > 2 ? 4 : 2, RPI = 64 / CPL;  // lanes of a staged row (16-byte chunks), rows a store
#pragma unroll
        for (int k = 0; k < 32 / RPI; ++k) {
          const int r = k * RPI + le / CPL, c = le % CPL;
          const uint4 v = *(const uint4*)(stage + r * 80 + c * 16);
          const int row = r0 + j * 32 + r, n = c0 + c * 32;
          const uint32_t off = c < FN && n < g.N ? (uint32_t)row * (uint32_t)(g.N >> 1) + (n >> 1) : 0x80000000u;
          __builtin_amdgcn_raw_buffer_store_b128((u32x4){v.x, v.y, v.z, v.w}, crs, (int)off, 0, 0);
        }
        // the wave's FN blocks of the row, code 0 for those past N
        const int row = r0 + j * 32 + er, blk = c0 >> 5;
        auto scale_at = [&](bool mine, int b) {
          return mine && row < rows && (b >> 3) < nslabs
                     ? (int)((uint32_t)(b >> 3) * (uint32_t)g.slab_c + (uint32_t)row * 8 + (b & 7))
                     : (int)0x80000000u;
        };
        if constexpr (FN == 4) {
          __builtin_amdgcn_raw_buffer_store_b32(codes, scr, scale_at(eh == 0, blk), 0, 0);
        } else if constexpr (FN == 3) {  // not at one place of a slab, nor always in one; the tiles reach the last slab's end
#pragma unroll
          for (int i = 0; i < 3; ++i)
            __builtin_amdgcn_raw_buffer_store_b8((uint8_t)(codes >> (8 * i)), scr, scale_at(eh == 0, blk + i), 0, 0);
        } else {  // tiles that end in the middle of the last slab write its unused bytes too, from the upper half
          const bool pad = eh == 1 && n0 + BN >= g.N && (n0 & 128) == 0;
          __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(eh ? 0 : codes), scr, scale_at(eh == 0 || pad, blk + eh * 4), 0, 0);
        }
      }
    } else {
      const __amdgpu_buffer_rsrc_t crs = __builtin_amdgcn_make_buffer_rsrc(
          (uint16_t*)g.C + m0 * g.N, 0, rows * g.N * 2, 0x00020000);
      // 32 rows of 32 kUnits columns at c0 + c, from the staged rows (16-bit)
      auto store_rows = [&](auto units, int j, int c) {
        constexpr int CPL = 4 * decltype(units)::value, RPI = 64 / CPL;  // 16-byte chunks of a row, rows a store
#pragma unroll
        for (int k = 0; k < 32 / RPI; ++k) {
          const int r = k * RPI + le / CPL, n = c0 + c + le % CPL * 8;
          const uint4 v = *(const uint4*)(stage + r * PITCH + le % CPL * 16);
          const uint32_t off = n < g.N ? ((uint32_t)(r0 + j * 32 + r) * (uint32_t)g.N + n) * 2 : 0x80000000u;
          __builtin_amdgcn_raw_buffer_store_b128((u32x4){v.x, v.y, v.z, v.w}, crs, (int)off, 0, 2);
        }
      };
      auto pack8 = [&](const float (&y)[8]) {
        return make_uint4(pack16x2<kBf16>(y[0], y[1]), pack16x2<kBf16>(y[2], y[3]), pack16x2<kBf16>(y[4], y[5]),
                          pack16x2<kBf16>(y[6], y[7]));
      };
      if constexpr (kEpi == kResidual) {
        const __amdgpu_buffer_rsrc_t rrs = __builtin_amdgcn_make_buffer_rsrc(
            (uint16_t*)g.residual + m0 * g.ldr, 0, (int)(((rows - 1) * g.ldr + g.N) * 2), 0x00020000);
        // a unit's fp32 rows through the staging area: 4 lanes a row, 16 rows a pass
        const int rr = le >> 2, rc = (le & 3) * 8;
#pragma unroll
        for (int i = 0; i < FN; ++i) {
          const int n = c0 + i * 32 + rc;
          float gt[8], b[2][8];
          side8(1024, i * 32 + rc, gt);
#pragma unroll
          for (int p = 0; p < 2; ++p) side8(0, i * 32 + 16 * p + 8 * eh, b[p]);
          u32x4 x[FM][2];
#pragma unroll
          for (int j = 0; j < FM; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t off =
                  n < g.N ? ((uint32_t)(r0 + j * 32 + k * 16 + rr) * (uint32_t)g.ldr + n) * 2 : 0x80000000u;
              x[j][k] = __builtin_amdgcn_raw_buffer_load_b128(rrs, (int)off, 0, 0);
            }
#pragma unroll
          for (int j = 0; j < FM; ++j) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              float y[8];
              columns(i, j, p, y);
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] += b[p][e];
              float4* s = (float4*)(stage + er * PITCH + (16 * p + 8 * eh) * 4);
              s[0] = make_float4(y[0], y[1], y[2], y[3]);
              s[1] = make_float4(y[4], y[5], y[6], y[7]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float4* s = (const float4*)(stage + (k * 16 + rr) * PITCH + rc * 4);
              const float4 a = s[0], c = s[1];
              float y[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint32_t r = x[j][k][e >> 1];
                y[e] = __builtin_fmaf(y[e], gt[e], e & 1 ? hi16<kBf16>(r) : lo16<kBf16>(r));
              }
              const uint4 v = pack8(y);
              const uint32_t off =
                  n < g.N ? ((uint32_t)(r0 + j * 32 + k * 16 + rr) * (uint32_t)g.N + n) * 2 : 0x80000000u;
              __builtin_amdgcn_raw_buffer_store_b128((u32x4){v.x, v.y, v.z, v.w}, crs, (int)off, 0, 2);
            }
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < FN; i += 2) {
          const int units = i + 1 < FN ? 2 : 1;
          float b[2][2][8];
#pragma unroll
          for (int u = 0; u < units; ++u)
#pragma unroll
            for (int p = 0; p < 2; ++p) side8(0, (i + u) * 32 + 16 * p + 8 * eh, b[u][p]);
#pragma unroll
          for (int j = 0; j < FM; ++j) {
#pragma unroll
            for (int u = 0; u < units; ++u)
#pragma unroll
              for (int p = 0; p < 2; ++p) {
                float y[8];
                columns(i + u, j, p, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  y[e] += b[u][p][e];
                  if constexpr (kEpi == kGelu) y[e] = gelu_tanh(y[e]);
                }
                *(uint4*)(stage + er * PITCH + u * 64 + p * 32 + eh * 16) = pack8(y);
              }
            if (units == 2)
              store_rows(IC<2>{}, j, i * 32);
            else
              store_rows(IC<1>{}, j, i * 32);
          }
        }
      }
    }
  };

  auto column_of = [&](int b) { return b < count ? tile_origin<BM, BN, kMainRows, kRest>(plan, b).n0 : 0; };
  load_tile(first);
  load_side(column_of(first), 0);
  int n_next = column_of(first + P);
#pragma unroll
  for (int s = 0; s < S; ++s) {
    aim();
#pragma unroll
    for (int d = 0; d < IA; ++d) load_a(d, lds0 + s * SLAB);
#pragma unroll
    for (int d = 0; d <= IW; ++d) load_w(d, lds0 + s * SLAB);
  }
  wait_vmcnt<(S - 2) * (IA + IW + 1)>();  // the first two slabs
  block_barrier();
#pragma unroll
  for (int j = 0; j < FM; ++j) read_a(j, 0);
#pragma unroll
  for (int i = 0; i < FA; ++i) read_w(i, 0);
  read_scales(0);
  for (int b = first; b < count; b += P) {
    const MxOrigin o = tile_origin<BM, BN, kMainRows, kRest>(plan, b);
    // in a tile's first slab the last epilogue's stores lie behind those loads too (none before the first tile, whose
    // first two slabs have landed)
    aim();
    slab_step(std::true_type{}, IC<kCounts.next_slab_first()>{}, n_next);
    for (int k = 1; k < nk; ++k) {
      aim();
      slab_step(std::false_type{}, IC<kCounts.next_slab()>{}, 0);
    }
    if constexpr (kCounts.side_waits()) {
      if (nk == 1) {  // no wait since this tile's bias and gate were loaded covers them
        wait_vmcnt<kCounts.side()>();
        block_barrier();
      }
    }
    epilogue(o.m0, o.n0);
    side_at = 2048 - side_at;
    n_next = column_of(b + 2 * P);
  }
  wait_vmcnt<0>();  // no load into LDS outlives the workgroup
}

constexpr int kTileLds = 160 * 1024 - 4096 - 4 * kStageBytes;  // for the ring

// F1: units of a rest tile's rows, 0 without a rest.
template <bool kBf16, int kEpi, int FM, int FN, int F1>
__global__ __launch_bounds__(256, 1) void mxfp4_gemm_tiles(MxGemmArgs g, MxTilePlan plan) {
  constexpr int S = kTileLds / tiles_lds(FM, FN) < 4 ? kTileLds / tiles_lds(FM, FN) : 4;
  static_assert(F1 <= FM, "rest tiles are no taller");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S * tiles_lds(FM, FN)];
  __shared__ __attribute__((aligned(1024))) uint8_t side[4096];  // bias and gate of this tile and the next
  __shared__ __attribute__((aligned(16))) uint8_t stage[4 * kStageBytes];
  run_tiles<kBf16, kEpi, FM, FN, S, 64 * FM, false>(g, plan, blockIdx.x, gridDim.x, plan.main, lds, side, stage);
  if constexpr (F1 > 0) {
    constexpr int S1 = S * tiles_lds(FM, FN) / tiles_lds(F1, FN);
    block_barrier();  // every wave has left the last main tile
    // on in the order of workgroups: those without a tile in the main tiles' last round come first
    const int P = gridDim.x, at = ((int)blockIdx.x - plan.main % P + P) % P;
    run_tiles<kBf16, kEpi, F1, FN, S1, 64 * FM, true>(g, plan, at < plan.rest_wgs ? at : plan.rest, plan.rest_wgs, plan.rest,
                                                      lds, side, stage);
  }
}

template <bool kBf16, int kEpi, int FM, int FN, int F1>
hipError_t launch_tiles(const MxGemmArgs& g, const MxTilePlan& p, hipStream_t st) {
  const int n = p.main + p.rest, cus = device_cus();
  hipLaunchKernelGGL((mxfp4_gemm_tiles<kBf16, kEpi, FM, FN, F1>), dim3((unsigned)(n < cus ? n : cus)), dim3(256), 0, st, g, p);
  return hipGetLastError();
}

// Few rows: a workgroup takes 32 NU columns of 32 MU rows and its waves share K, slab after slab (wave w the slabs w,
// w + W, ...), each with a ring of S slabs in LDS of its own, so that no barrier holds up the loads, which are what
// these calls are bound by. The partial sums go through LDS and are added in the order of the waves. W from HBM, calls in a
// loop with the gaps between launches, against the tile kernels: 1 x 4096 x 12288 12.5 -> 8.4 us (3.2 TB/s), 64 x 5120 x
// 5120 16.3 -> 8.4, 64 x 13824 x 5120 31 -> 17, 64 x 5120 x 13824 18 -> 14.7. The kernels alone, W from HBM and from the
// last-level cache: 7.6 and 5.6, 8.3 and 6.1, 14.9 and 11.8, 13.4 (216 workgroups on 256 CUs) and 10.5.
template <bool kBf16, int kEpi, int NU, int MU, int W, int S>
__global__ __launch_bounds__(64 * W) void mxfp4_gemm_rows(MxGemmArgs g) {
  constexpr int RB = 128, kUnit = 32 * RB + 256;   // a unit's rows, then their scales
  constexpr int SLAB = (NU + MU) * kUnit;          // W units, then A units
  constexpr int LOADS = (NU + MU) * 5;            // of a slab
  constexpr int BN = 32 * NU, PITCH = BN + 4;      // floats of a row of partial sums
  static_assert(W * S * SLAB <= 160 * 1024 && (S - 1) * LOADS < 64, "LDS, vmcnt range");
  static_assert(W * MU * 32 * PITCH * 4 <= W * S * SLAB, "partial sums");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[W * S * SLAB];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int Kb = g.K >> 1, nk = (g.K + 255) >> 8;
  const int n0 = blockIdx.x * BN;
  const int64_t m0 = (int64_t)blockIdx.y * (32 * MU);
  const int rows = (int)min((int64_t)(32 * MU), g.M - m0), cols = min(BN, g.N - n0);
  // operands and scales of W (0) and A (1): their starts and the bytes from there on (rows past the last load zeros)
  const uint8_t* const op[2] = {(const uint8_t*)g.W + (int64_t)n0 * Kb, (const uint8_t*)g.A + m0 * Kb};
  const uint8_t* const sp[2] = {(const uint8_t*)g.scales_b + (int64_t)n0 * 8, (const uint8_t*)g.scales_a + m0 * 8};
  const int op_bytes[2] = {cols * Kb, rows * Kb};
  const int sp_bytes[2] = {(int)((nk - 1) * g.slab_b + (g.N - n0) * 8), (int)((nk - 1) * g.slab_a + (g.M - m0) * 8)};
  const uint32_t lds0 = lds_u32((lds_void*)lds) + wave * (S * SLAB);
  uint32_t off[4];  // of the four loads of a unit: 8 rows each, chunk c of row r at c ^ swz(r)
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int row = d * 8 + (lane >> 3);
    off[d] = (uint32_t)row * (uint32_t)Kb + (uint32_t)(((lane & 7) ^ (row & 7) ^ (d & 1)) * 16);
  }
  auto load = [&](int k, int slot) {  // slab k; past the last from empty ranges, so that every slab counts as many loads
    const uint32_t dst = lds0 + slot * SLAB;
    const bool in = k < nk;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)op[o], 0, in ? op_bytes[o] : 0, 0x00020000);
      const __amdgpu_buffer_rsrc_t ss = __builtin_amdgcn_make_buffer_rsrc((void*)sp[o], 0, in ? sp_bytes[o] : 0, 0x00020000);
      const uint32_t so = in ? (uint32_t)k * (uint32_t)(o ? g.slab_a : g.slab_b) : 0u;
#pragma unroll
      for (int i = 0; i < (o ? MU : NU); ++i) {
        const uint32_t to = dst + ((o ? NU : 0) + i) * kUnit;
#pragma unroll
        for (int d = 0; d < 4; ++d) dma_buf16(to + d * 1024, off[d] + (uint32_t)(i * 32) * (uint32_t)Kb, rs, in ? k * RB : 0);
        dma_buf4(to + 4096, (uint32_t)(lane * 4 + i * 256) + so, ss);
      }
    }
  };
  const int frow = lane & 31, half = lane >> 5, fsw = (frow & 7) ^ ((frow >> 3) & 1);
  v16f acc[NU][MU];
#pragma unroll
  for (int i = 0; i < NU; ++i)
#pragma unroll
    for (int j = 0; j < MU; ++j) acc[i][j] = (v16f){};
#pragma unroll
  for (int s = 0; s < S; ++s) load(wave + s * W, s);
  int slot = 0;
  for (int k = wave; k < nk; k += W) {
    wait_vmcnt<(S - 1) * LOADS>();
    asm volatile("" ::: "memory");
    const uint8_t* src = lds + wave * (S * SLAB) + slot * SLAB;
    v4i f[NU + MU][4];
    int sc[NU + MU];
#pragma unroll
    for (int u = 0; u < NU + MU; ++u) {
      const uint8_t* a = src + u * kUnit;
      sc[u] = *(const int*)(a + 4096 + frow * 8 + half * 4);
#pragma unroll
      for (int t = 0; t < 4; ++t) f[u][t] = *(const v4i*)(a + frow * RB + ((4 * half + t) ^ fsw) * 16);
    }
    wait_lgkm0();  // the slot has been read
    asm volatile("" ::: "memory");
    load(k + S * W, slot);
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int j = 0; j < MU; ++j) {
        v16f& c = acc[i][j];
        c = mfma_fp4<0>(f[i][0], f[NU + j][0], c, sc[i], sc[NU + j]);
        c = mfma_fp4<1>(f[i][1], f[NU + j][1], c, sc[i], sc[NU + j]);
        c = mfma_fp4<2>(f[i][2], f[NU + j][2], c, sc[i], sc[NU + j]);
        c = mfma_fp4<3>(f[i][3], f[NU + j][3], c, sc[i], sc[NU + j]);
      }
    slot = slot + 1 == S ? 0 : slot + 1;
  }
  wait_vmcnt<0>();  // nothing is on its way into LDS any more
  block_barrier();
  float* part = (float*)lds;
#pragma unroll
  for (int i = 0; i < NU; ++i)
#pragma unroll
    for (int j = 0; j < MU; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(float4*)(part + ((wave * MU + j) * 32 + frow) * PITCH + i * 32 + 8 * q + 4 * half) =
            make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
  __syncthreads();
  // eight columns of a row a thread, a quad of threads an MXFP4 block
  auto row8 = [&](const void* p, int64_t at, float (&v)[8]) {
    const uint4 x = *(const uint4*)((const uint16_t*)p + at);
    const uint32_t d[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = lo16<kBf16>(d[e]);
      v[2 * e + 1] = hi16<kBf16>(d[e]);
    }
  };
  for (int x = threadIdx.x; x < 32 * MU * 4 * NU; x += 64 * W) {
    const int r = x / (4 * NU), c = x % (4 * NU) * 8;
    float y[8] = {};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float4* s = (const float4*)(part + (w * MU * 32 + r) * PITCH + c);
      const float4 a = s[0], b = s[1];
      y[0] += a.x, y[1] += a.y, y[2] += a.z, y[3] += a.w, y[4] += b.x, y[5] += b.y, y[6] += b.z, y[7] += b.w;
    }
    const int n = n0 + c;
    const int64_t m = m0 + r;
    const bool in = m < g.M && n < g.N;
    if (in && g.bias) {
      float b[8];
      row8(g.bias, n, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] += b[e];
    }
    if constexpr (kEpi == kGelu || kEpi == kGeluQuant) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = gelu_tanh(y[e]);
    }
    if constexpr (kEpi == kGeluQuant) {
      const uint32_t code = mx_code(quad_max_u32(abs_max8(y)));
      if (!in) continue;
      *(uint32_t*)((uint8_t*)g.C + m * (g.N >> 1) + (n >> 1)) = mx_pack8(y, mx_scale(code));
      uint8_t* s = (uint8_t*)g.out_s + m * 8;
      const int blk = n >> 5;
      if ((c & 31) == 0) s[(blk >> 3) * g.slab_c + (blk & 7)] = (uint8_t)code;
      if ((c & 31) == 8 && blk * 32 + 32 == g.N)  // the last slab's unused bytes
        for (int b = blk + 1; b & 7; ++b) s[(b >> 3) * g.slab_c + (b & 7)] = 0;
    } else {
      if (!in) continue;
      if constexpr (kEpi == kResidual) {
        float x[8], gt[8];
        row8(g.residual, m * g.ldr + n, x);
        row8(g.gate, n, gt);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf(y[e], gt[e], x[e]);
      }
      *(uint4*)((uint16_t*)g.C + m * g.N + n) = make_uint4(pack16x2<kBf16>(y[0], y[1]), pack16x2<kBf16>(y[2], y[3]),
                                                           pack16x2<kBf16>(y[4], y[5]), pack16x2<kBf16>(y[6], y[7]));
    }
  }
}

template <bool kBf16, int kEpi, int NU, int MU, int W, int S>
hipError_t launch_rows(const MxGemmArgs& g, hipStream_t st) {
  const dim3 grid((unsigned)((g.N + 32 * NU - 1) / (32 * NU)), (unsigned)((g.M + 32 * MU - 1) / (32 * MU)));
  hipLaunchKernelGGL((mxfp4_gemm_rows<kBf16, kEpi, NU, MU, W, S>), grid, dim3(64 * W), 0, st, g);
  return hipGetLastError();
}

// The tile shape of a call: the one whose tiles keep the busiest CU busy for the shortest time, in units of a 256 x 256
// tile's. What the others take of it (10800 x 5120 x 15360, where all CUs are busy and the clock is what the power
// allows, and 128 x 5120 x 5120 against 64 x 13824 x 5120, where neither holds: within 5 % of each other): operand
// bytes and instructions per MFMA grow as tiles shrink. 256 x 192 and 256 x 128 tiles win at no shape of the block.
enum TileShape : int { k256x256 = 0, k128x256, k128x192, k128x128, k64x128 };
constexpr struct {
  int bm, bn;
  float cost;
} kTileShapes[] = {{256, 256, 1.0f}, {128, 256, 0.6f}, {128, 192, 0.47f}, {128, 128, 0.345f}, {64, 128, 0.25f}};
constexpr float kRestCost = 0.45f;  // a 64 x 256 rest tile

struct TileChoice {
  TileShape shape;
  MxTilePlan plan;
};
TileChoice choose_tiles(int64_t M, int N, bool quant, int cus) {
  TileChoice best = {};
  float best_cost = 0.f;
  auto offer = [&](TileShape s, const MxTilePlan& p, float cost) {
    if (best_cost != 0.f && cost >= best_cost) return;
    best = {s, p};
    best_cost = cost;
  };
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  for (int s = k256x256; s <= k64x128; ++s) {
    MxTilePlan p = {};
    p.tiles_m = (int)up(M, kTileShapes[s].bm);
    // 192 columns end in the middle of a scale slab, whose unused bytes are some tile's to write (with MXFP4 output, 347 x
    // 5120 x 13824 33.8 us without this shape, 26.8 with it; 700 x 4096 x 6144 24.9 and 19.1)
    p.tiles_n = (int)up(quant && s == k128x192 ? up(N, 256) * 256 : N, kTileShapes[s].bn);
    p.main = p.tiles_m * p.tiles_n;
    offer((TileShape)s, p, kTileShapes[s].cost * (float)up(p.main, cus));
  }
  // 256 x 256 tiles without a short last row of them: its rows go to rest tiles, which start on the CUs that the last
  // round of main tiles leaves idle (3120 x 4096 x 16384: 119 -> 112 us)
  if (M > 256 && M % 256 != 0) {
    MxTilePlan p = {};
    p.tiles_m = (int)(M / 256);
    p.tiles_n = (int)up(N, 256);
    p.main = p.tiles_m * p.tiles_n;
    p.rest = (int)up(M % 256, 64) * p.tiles_n;
    const int rounds = p.main / cus, odd = p.main % cus, idle = cus - odd;
    // two rest tiles take no longer than a main one (3120 x 5120 x 5120, 240 main tiles and 20: 54 -> 47 us)
    const bool twice = odd && p.rest <= 2 * idle;
    p.rest_wgs = twice ? std::min(idle, p.rest) : std::min(cus, p.main + p.rest);
    const float early = (float)rounds + kRestCost * (float)up(p.rest, twice ? idle : cus);
    const float late = odd ? (float)(rounds + 1) + (twice ? 0.f : kRestCost * (float)up(p.rest - idle, cus)) : 0.f;
    offer(k256x256, p, early > late ? early : late);
  }
  return best;
}

template <bool kBf16, int kEpi>
hipError_t launch_epi(const MxGemmArgs& g, hipStream_t st) {
  // Up to 128 rows whose units of 32 x 32 are few: a workgroup of two waves each (34 KB, four of them a CU). More of
  // them would read the activations too often; up to 64 rows then take 64 x 64 a workgroup of four waves. (128 x 5120
  // x 5120, 640 units: 11.9 us against the tiles' 15.3; 64 x 5120 x 13824, 864: 17.7 against 14.7 of the second kind;
  // 128 x 5120 x 15360, 1920: 28 against the tiles' 19.)
  const int64_t units = (int64_t)((g.N + 31) / 32) * ((g.M + 31) / 32);
  if (g.M <= 128 && units * 2 <= 5 * device_cus()) return launch_rows<kBf16, kEpi, 1, 1, 2, 2>(g, st);
  if (g.M <= 64) return launch_rows<kBf16, kEpi, 2, 2, 4, 2>(g, st);
  const TileChoice c = choose_tiles(g.M, g.N, kEpi == kGeluQuant, device_cus());
  switch (c.shape) {
    case k256x256: return launch_tiles<kBf16, kEpi, 4, 4, 1>(g, c.plan, st);
    case k128x256: return launch_tiles<kBf16, kEpi, 2, 4, 0>(g, c.plan, st);
    case k128x192: return launch_tiles<kBf16, kEpi, 2, 3, 0>(g, c.plan, st);
    case k128x128: return launch_tiles<kBf16, kEpi, 2, 2, 0>(g, c.plan, st);
    case k64x128: return launch_tiles<kBf16, kEpi, 1, 2, 0>(g, c.plan, st);
  }
  return hipErrorInvalidValue;
}

template <bool kBf16>
hipError_t launch_t(const MxGemmArgs& g, hipStream_t st) {
  if (g.out_s) return launch_epi<kBf16, kGeluQuant>(g, st);
  if (g.residual) return launch_epi<kBf16, kResidual>(g, st);
  if (g.gelu) return launch_epi<kBf16, kGelu>(g, st);
  return launch_epi<kBf16, kPlain>(g, st);
}

}  // namespace

hipError_t launch_mxfp4_gemm(const MxGemmArgs& g, hipStream_t st) {
  return g.bf16 ? launch_t<true>(g, st) : launch_t<false>(g, st);
}

}  // namespace joy
