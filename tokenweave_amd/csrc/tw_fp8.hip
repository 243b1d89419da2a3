// Rows to e4m3 codes with a scale for 128 channels, and the product of such rows with a weight of
// e4m3 codes that has a scale for each block of 128 x 128.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "tw_activation.h"
#include "tw_common.h"
#include "tw_store.h"

namespace tw {

namespace {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) uint8_t lds_u8_t;
typedef __attribute__((address_space(3))) const u32x4_t lds_chunk_t;
typedef __attribute__((address_space(3))) const float lds_f32_t;

constexpr int GROUP = TW_FP8_GROUP;

// ---------------------------------------------------------------------------
// Codes
//
// A group of 128 channels is 16 lanes of 8: their largest magnitude by four exchanges, their codes as 8 bytes a lane.
// A workgroup takes 16 rows of one group, its neighbours the next groups of the same rows: whole lines are read, and
// the 16 scales leave together where the scales' rows are adjacent.  Bound by memory: act(gate) * up of [8192, 2 x 3584] in
// bf16 31 us (148 MB, 4.8 TB/s); 1001 x 3696 in fp16 4.6 us, 32 x 8192 3.6: a launch and one trip to memory.
//
// K % 8 != 0, or rows that do not begin on 16 bytes (VEC = false): element by element, bound by the instructions of 2-byte
// loads and 1-byte stores: 8192 x 7161 in bf16 114 us (1.6 TB/s; 7168 wide 41), fp32 146 (50), gated 8192 x 3581 95 (33),
// 1001 x 3695 in fp16 10.0 (4.7), 32 x 8191 3.5.
// ---------------------------------------------------------------------------
constexpr int QUANT_THREADS = 256;
constexpr int QUANT_ROWS = QUANT_THREADS / 16;

struct QuantArgs {
  uint8_t* out;
  float* scales;
  const void* input;
  int64_t scale_row, scale_group, ld_in;
  int M, K, groups, act;
};

template <int DTYPE>
__device__ __forceinline__ float load_one(const void* p, int64_t i) {
  if (DTYPE == TW_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (DTYPE == TW_DTYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
  return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
}

// Eight values from element `at` on, the first `n` of them; the others are zeros.  VEC: all or none, and 16-byte
// aligned.
template <int DTYPE, bool VEC>
__device__ __forceinline__ void load_eight(float (&v)[8], const void* p, int64_t at, int n) {
  if (!VEC) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? load_one<DTYPE>(p, at + e) : 0.0f;
    return;
  }
  if (n < 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
  } else if (DTYPE == TW_DTYPE_F32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 x = q[0], y = q[1];
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (DTYPE == TW_DTYPE_F16) {
        const f16x2_t h = __builtin_bit_cast(f16x2_t, w[e]);
        v[2 * e] = (float)h.x, v[2 * e + 1] = (float)h.y;
      } else {
        v[2 * e] = __uint_as_float(w[e] << 16), v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      }
    }
  }
}

// y / s as a float that rounds to the same e4m3 code as the exact quotient.  `inverse` is 1 / s; one correction makes
// q the nearest float.  That may lie on the border of two codes (its low 19 bits are then zero; also below the least
// normal code, whose borders have fewer bits) where the quotient does not: there q goes towards zero to the odd
// neighbour or keeps its place with the lowest bit set, as the remainder says.
__device__ __forceinline__ float quotient(float y, float s, float inverse) {
  float q = y * inverse;
  q = __fmaf_rn(__fmaf_rn(-q, s, y), inverse, q);
  if ((__float_as_uint(q) & 0x7ffffu) == 0) {
    const float rest = __fmaf_rn(-q, s, y);
    if (rest != 0.0f) {
      uint32_t bits = __float_as_uint(q);
      if ((__float_as_uint(rest) ^ __float_as_uint(y)) >> 31) bits -= 1;  // |q| is the larger one; bits end in zeros
      q = __uint_as_float(bits | 1u);
    }
  }
  return q;
}

template <int DTYPE, bool GATED, bool VEC>
__global__ __launch_bounds__(QUANT_THREADS) void quant_fp8_groups_kernel(QuantArgs w) {
  const int unit = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int group = blockIdx.x % w.groups, row = blockIdx.x / w.groups * QUANT_ROWS + unit;
  if (row >= w.M) return;
  const int c = group * GROUP + lane * 8, n = min(max(w.K - c, 0), 8);
  const int64_t at = row * w.ld_in + c;
  float y[8];
  load_eight<DTYPE, VEC>(y, w.input, at, n);
  if (GATED) {
    float u[8];
    load_eight<DTYPE, VEC>(u, w.input, at + w.K, n);
    with_activation(w.act, [&](auto act) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = activation<act()>(y[e]) * u[e];
    });
  }
  // as whole numbers magnitudes are in order, infinities and NaN above all others
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(y[e]) & 0x7fffffffu);
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, x, 16));
  const float largest = __uint_as_float(max(most, __float_as_uint(1e-10f)));
  const float s = __fdiv_rn(largest, 448.0f);
  if (lane == 0) w.scales[row * w.scale_row + group * w.scale_group] = s;
  uint32_t code[2] = {0x7f7f7f7fu, 0x7f7f7f7fu};
  if (most < 0x7f800000u) {
    const float inverse = __frcp_rn(s);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = quotient(y[e], s, inverse);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
      code[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], v, true);
    }
  }
  uint8_t* to = w.out + (int64_t)row * w.K + c;
  if (VEC) {
    if (n == 8) *reinterpret_cast<uint2*>(to) = make_uint2(code[0], code[1]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) to[e] = (uint8_t)(code[e >> 2] >> (8 * (e & 3)));
  }
}

template <int DTYPE>
void launch_quant(const QuantArgs& w, bool vec, int64_t grid, hipStream_t hs) {
  auto go = [&](auto kernel) { launch_kernel(kernel, dim3((unsigned)grid), dim3(QUANT_THREADS), 0, hs, w); };
  if (w.act >= 0) vec ? go(quant_fp8_groups_kernel<DTYPE, true, true>) : go(quant_fp8_groups_kernel<DTYPE, true, false>);
  else vec ? go(quant_fp8_groups_kernel<DTYPE, false, true>) : go(quant_fp8_groups_kernel<DTYPE, false, false>);
}

// ---------------------------------------------------------------------------
// The product.  A slab is one block of 128 of the inner dimension: 128 bytes a row, one matrix instruction of
// 16 x 16 x 128 (two of 32 x 32 x 64) without a running sum, whose result is added to the fp32 sums with the product
// of both scales.  Slabs lie in LDS as the bf16 kernels' do (128-byte rows, 16-byte chunk c of row r at c ^ key(r)).  The
// order of the inner dimension inside an instruction is the same for both operands and otherwise free: a lane takes
// chunks q and q + 4 of a row.
//
// The instruction adds aligned eights of products at 13 bits below the largest one's exponent, and those sums in fp32
// (measured; the tests look at it): fewer bits than fp32 for a sum of eight, taken for the rate of this instruction.  A
// code itself stands for its value to 4 bits, and fp16 results of 3696 channels are off by 2.1e-4 in the mean square, as
// those of sums in fp32 throughout.
// ---------------------------------------------------------------------------
constexpr int ROWB = 128;
[[maybe_unused]] constexpr uint32_t OUT_OF_RANGE = 0x80000000u;
constexpr int64_t BLOCK_MAX_K = 1 << 22;  // a tile's rows span at most 1 GiB
constexpr int64_t BLOCK_WIDE_LDC = 1 << 22;  // 256 rows of the output, where they are stored 16 bytes a lane: 2 GiB

constexpr int64_t BLOCK_MAX_SCALE_ROW = 1 << 20;  // 32-bit offsets of a tile's scales

struct BlockArgs {
  uint16_t* out;
  const uint8_t *a, *b;
  const float *a_scales, *b_scales;
  int64_t scale_row, scale_block, ldc;
  int M, N, K, half_out, tiles_m, tiles_n, cols;
  int form;  // StoreForm, tile kernel
  float* sums;     // tile kernel, K divided: [parts][M][N], `per` slabs a part
  int parts, per;
};

[[maybe_unused]] __device__ __forceinline__ uint32_t pack_out(float lo, float hi, int half_out) {
  const f32x2_t v = {lo, hi};
  const uint32_t half = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
  const uint32_t brain = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
  return half_out ? half : brain;
}

#ifdef __HIP_DEVICE_COMPILE__
// One fp32 a lane, `offset` bytes behind `from`, to LDS.  (A buffer load: behind a global load to LDS the compiler makes
// every wait for an LDS read a wait for all of them, and for all loads.)
__device__ __forceinline__ void load_scales(const float* from, uint32_t offset, lds_u8_t* to) {
  const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(from), 0, 0x7fffffffu, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (lds_void_t*)to, 4, offset, 0, 0, 0);
}
__device__ __forceinline__ i32x8_t fragment(const lds_u8_t* p, const lds_u8_t* q) {
  const u32x4_t x = *(lds_chunk_t*)p, y = *(lds_chunk_t*)q;
  return i32x8_t{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, (int)y.z, (int)y.w};
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
#endif

// Few rows: bound by reading b once.  As in the bf16 K-split kernel four waves share the inner dimension, wave w takes
// the slabs w, w + 4, ..., each brings its own slabs of both operands and the rows' scales into LDS of its own, and the
// four sums meet at the end as ((w0 + w1) + w2) + w3.  All scales come through LDS: a scalar or vector load under way
// makes the compiler wait for more than a slab needs ([1, 3584] x [8192, 3584]^T 8.2 -> 6.7 us, [96, 8192] x [7168, 8192]^T
// 24.5 -> 19.8).
//
// [1, 8192] x [7168, 8192]^T 10.6 us (59 MB, 5.5 TB/s), 32 rows 11.8, 64 rows 12.9 (4.7 TB/s), 96 rows 17.6 to 19.8: from
// 65 rows on a is read by two row tiles, and what bounds a compute unit is the 50 GB/s of all its lines (0.9 MB there).
// K cut into quarters over 64 x 128 tiles of 448 workgroups takes 16.3 us, and another launch to add them.
constexpr int SPLIT_WAVES = 4;
constexpr int SPLIT_THREADS = SPLIT_WAVES * 64;
constexpr int split_stage(int mt, int nt) { return 32 * (mt + nt) * ROWB + 256; }
constexpr int split_wave(int mt, int nt, int stages) { return stages * split_stage(mt, nt) + 512; }
constexpr int split_lds(int mt, int nt, int stages) {
  const int slabs = SPLIT_WAVES * split_wave(mt, nt, stages), sums = SPLIT_WAVES * 32 * mt * (32 * nt * 4 + 16);
  return slabs > sums ? slabs : sums;
}

template <int MT, int NT, int STAGES, int LA>
__global__ __launch_bounds__(SPLIT_THREADS) void gemm_fp8_block_split_kernel(BlockArgs w) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int RA = 32 * MT, RB = 32 * NT, LB = RB / 8, ROWS = 8 * LA, STAGE = split_stage(MT, NT);
  constexpr int LOADS = LA + LB + 1;
  static_assert(ROWS <= RA && RA <= 64, "one load of 64 lanes brings the rows' scales");
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, lhi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = w.K, nk = (K + GROUP - 1) / GROUP, tail_chunks = (K % GROUP) / 16;
  const bool even = ((lane & 7) ^ (lane >> 4)) < tail_chunks, odd = ((lane & 7) ^ (lane >> 4) ^ 4) < tail_chunks;
  uint32_t v[LA > LB ? LA : LB], roff[4];
#pragma unroll
  for (int j = 0; j < (LA > LB ? LA : LB); ++j)
    v[j] = (uint32_t)(j * 8 + (lane >> 3)) * (uint32_t)K + (((lane & 7) ^ (((j & 1) << 2) | (lane >> 4))) << 4);
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) roff[kk] = l32 * ROWB + ((((kk << 1) | lhi) ^ ((l32 >> 1) & 7)) << 4);
  // the wave's slabs, and the weight's scales of 64 of them, for both blocks that a tile may touch
  uint8_t* const mine = lds + wave * split_wave(MT, NT, STAGES);
  lds_u8_t* const block_scales = (lds_u8_t*)mine + STAGES * STAGE;

  const int num_tiles = w.tiles_m * w.tiles_n;
  for (int t = blockIdx.x; t < num_tiles; t += gridDim.x) {
    // every XCD a contiguous range of tiles, the row tiles of one column range next to each other
    int pid = t;
    const int per_xcd = num_tiles / 8;
    if (t < per_xcd * 8) pid = (t & 7) * per_xcd + (t >> 3);
    const int m0 = pid % w.tiles_m * ROWS, n0 = pid / w.tiles_m * w.cols;
    const int rows = min(w.M - m0, ROWS);
    const __amdgpu_buffer_rsrc_t da = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(w.a) + (size_t)m0 * K, 0, (uint32_t)rows * (uint32_t)K, 0x00020000);
    const __amdgpu_buffer_rsrc_t db = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(w.b) + (size_t)n0 * K, 0, (uint32_t)min(w.N - n0, w.cols) * (uint32_t)K, 0x00020000);
    // a row's scales, one for each lane that has a row
    const float* const scales = w.a_scales + (int64_t)m0 * w.scale_row;
    const uint32_t my_scale = (uint32_t)min(lane, rows - 1) * (uint32_t)w.scale_row * 4u;
    // columns before `border` belong to the first of the two weight blocks that a tile may touch
    const float* const sb = w.b_scales + (int64_t)(n0 / GROUP) * nk;
    const int border = GROUP - n0 % GROUP;
    const int64_t second = n0 / GROUP + 1 < (w.N + GROUP - 1) / GROUP ? nk : 0;
    auto fetch_blocks = [&](int from) {
      const uint32_t at = (uint32_t)min(from + SPLIT_WAVES * lane, nk - 1) * 4u;
      load_scales(sb, at, block_scales);
      load_scales(sb + second, at, block_scales + 256);
    };
    fetch_blocks(wave);
    uint32_t turn = 0;

    f32x16_t acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    int next = wave;
    uint32_t fill = 0, use = 0;
    auto issue = [&]() {
      const bool last = tail_chunks && next == nk - 1;
      uint8_t* s = mine + fill;
      const uint32_t koff = (uint32_t)next * ROWB;
#pragma unroll
      for (int j = 0; j < LB; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(db, (lds_void_t*)(s + RA * ROWB + j * 1024), 16,
                                                 !last || ((j & 1) ? odd : even) ? v[j] : OUT_OF_RANGE, koff, 0, 0);
#pragma unroll
      for (int j = 0; j < LA; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(da, (lds_void_t*)(s + j * 1024), 16,
                                                 !last || ((j & 1) ? odd : even) ? v[j] : OUT_OF_RANGE, koff, 0, 0);
      load_scales(scales + next * w.scale_block, my_scale, (lds_u8_t*)(s + (RA + RB) * ROWB));
      next += SPLIT_WAVES;
      fill = fill == (STAGES - 1) * STAGE ? 0 : fill + STAGE;
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
      if (next < nk) issue();
    for (int slab = wave; slab < nk; slab += SPLIT_WAVES, use = use == (STAGES - 1) * STAGE ? 0 : use + STAGE) {
      if (turn == 256) {
        fetch_blocks(slab);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        turn = 0;
      }
      if (next < nk) {
        issue();
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * LOADS) : "memory");
      } else if (STAGES == 3 && slab + SPLIT_WAVES < nk) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      const uint8_t* pa = mine + use;
      const uint8_t* pb = pa + RA * ROWB;
      f32x16_t part[MT][NT];
      i32x8_t fa[2][MT], fb[2][NT];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
          fb[h][j] = fragment((lds_u8_t*)pb + j * 32 * ROWB + roff[2 * h], (lds_u8_t*)pb + j * 32 * ROWB + roff[2 * h + 1]);
#pragma unroll
        for (int i = 0; i < MT; ++i)
          fa[h][i] = fragment((lds_u8_t*)pa + i * 32 * ROWB + roff[2 * h], (lds_u8_t*)pa + i * 32 * ROWB + roff[2 * h + 1]);
      }
      const float block0 = *(lds_f32_t*)(block_scales + turn), block1 = *(lds_f32_t*)(block_scales + 256 + turn);
      turn += 4;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
            part[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[h][j], fa[h][i], h ? part[i][j] : f32x16_t{}, 0,
                                                                         0, 0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float sa = *reinterpret_cast<const float*>(mine + use + (RA + RB) * ROWB + (i * 32 + l32) * 4);
        const float s0 = sa * block0, s1 = sa * block1;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float s = j * 32 + 8 * q + 4 * lhi < border ? s0 : s1;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = __fmaf_rn(part[i][j][4 * q + e], s, acc[i][j][4 * q + e]);
          }
      }
      // the fragments and scales are in registers: the loads issued next may overwrite this stage
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }

    // A wave without a slab has its block scales under way still: they must not land among the sums.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    // acc[i][j][4 q + e]: sum of out[m0 + i*32 + l32][n0 + j*32 + 8 q + 4 lhi + e]
    constexpr int PITCH = RB * 4 + 16;
    __syncthreads();
    uint8_t* const sums = lds + wave * (RA * PITCH);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4_t*>(sums + (i * 32 + l32) * PITCH + (j * 32 + 8 * q + 4 * lhi) * 4) =
              f32x4_t{acc[i][j][4 * q + 0], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __syncthreads();
    for (int g = tid; g < ROWS * RB / 4; g += SPLIT_THREADS) {
      const int m = g / (RB / 4), c = (g % (RB / 4)) * 4;
      if (m < rows && c < w.cols && n0 + c < w.N) {
        const uint8_t* p = lds + m * PITCH + c * 4;
        f32x4_t s = *reinterpret_cast<const f32x4_t*>(p);
#pragma unroll
        for (int x = 1; x < SPLIT_WAVES; ++x) s += *reinterpret_cast<const f32x4_t*>(p + x * (RA * PITCH));
        *reinterpret_cast<uint2*>(w.out + (size_t)(m0 + m) * w.ldc + n0 + c) =
            make_uint2(pack_out(s.x, s.y, w.half_out), pack_out(s.z, s.w, w.half_out));
      }
    }
    __syncthreads();  // the next tile's slabs overwrite the sums
  }
#endif
}

// More rows: eight waves, WM x (8 / WM) of them, each (16 TM) x (16 TN) of the output.  The sums cannot stay in
// accumulation registers, which vector instructions do not reach: two waves a SIMD of 256 registers each.
//
// A slab is TM rows of TN matrix instructions; what goes on beside them is placed by hand:
//  * behind each instruction the four multiply-adds of the one LAG earlier, whose results have arrived;
//  * a row's fragment of a is read from LDS one row ahead, the slab's fragments of b in the last row of the slab before,
//    each as its register has served;
//  * a barrier lies before a slab's last row.  It says that the next slab has arrived and, as all fragments of this one
//    are in registers, that its place in LDS is free: a's rows of the slab NA ahead go there;
//  * b's rows are all in registers a row into the slab.  Where LDS holds two slabs of them only, a second barrier says
//    so there, and those of the slab after the next set out most of a slab earlier than they otherwise could.
// Loads go out one per SPACE instructions: in a burst they hold up all waves, the unit's path to memory takes 64 bytes a
// cycle.
//
// [4096, 8192] x [7168, 8192]^T, us, one change at a time: left to the compiler 294; placed as above, two slabs 253; a's
// slab three ahead, b's by a barrier of its own and 256 x 224 tiles 205 to 214 by board (2 300 TFLOP/s; 8192^3 of the
// library with one scale a tensor 2 920).  In 256 x 256 tiles without the loads 211 of 253, without the multiply-adds 233,
// without both 184: the matrix cores themselves, at the clock that the board's power limit leaves.
// [1000, 3696] x [8192, 3696]^T 35.3 us: 256 tiles, a unit's 1.4 MB at its 50 GB/s, and 5 us that a single slab takes as
// well (8 bytes a lane and store: 39.2).
constexpr int WIDE_THREADS = 512;
template <int WM, int TM, int TN, int NA, int NB>
struct WideShape {
  static constexpr int WN = 8 / WM, BM = 16 * TM * WM, BN = 16 * TN * WN, PA = BM * ROWB;
  static constexpr int LA = BM / 64, LB = (BN + 63) / 64;  // loads of 8 rows a wave and slab
  static constexpr int PB = BN * ROWB;                     // (BN % 64 != 0: some waves' last load goes nowhere)
  static constexpr bool EARLY = NB < NA || NB == 2;        // b's rows by a barrier of their own
  static constexpr int AT_B = NA * PA, AT_S = AT_B + NB * PB, AT_NONE = AT_S + NA * BM * 4;
  static constexpr int LDS = AT_NONE + (BN % 64 ? 1024 : 0);
  // loads under way that a slab's barrier does not wait for: what was issued behind the next slab's
  static constexpr int PENDING = !EARLY ? (NA - 2) * (LA + LB + 1) : (NA - 2) * (LA + 1) + LB;
  static constexpr int LATE = EARLY ? LA + 1 : LA + LB + 1;  // loads that follow the barrier before the last row
  static constexpr int SPACE_LATE = EARLY ? 1 : TM * TN / LATE / 2 < 1 ? 1 : TM * TN / LATE / 2;
  static constexpr int SPACE_EARLY = (TM - 2) * TN / LB / 2 < 1 ? 1 : (TM - 2) * TN / LB / 2;
  static constexpr int TOTAL = TM * TN, LAG = TN < 3 ? TN : 3, RING = 4;  // results in registers
  static_assert(TOTAL % RING == 0 && LAG < RING, "an instruction's results have one place in every slab");
  static_assert(TM % 2 == 0 && BM % 64 == 0 && LDS <= 160 * 1024 && NA == 3 && NB >= 2 && NB <= 3, "shape");
  static_assert(EARLY ? TM > 2 && NB == 2 && (LATE - 1) * SPACE_LATE < 2 * TN && (LB - 1) * SPACE_EARLY < (TM - 2) * TN
                      : (LATE - 1) * SPACE_LATE < TM * TN, "every load has a place");
};

#ifdef __HIP_DEVICE_COMPILE__
__device__ __forceinline__ uint32_t after(uint32_t at, uint32_t panel, int n) {
  return at == (n - 1) * panel ? 0u : at + panel;
}
#endif

// TAIL: the last slab is a partial one, whose chunks past K must arrive as zeros.  SPLIT: `parts` workgroups share a tile's
// slabs and leave fp32 sums, which block_join_kernel adds in order.
template <int WM, int TM, int TN, int NA, int NB, bool TAIL, bool SPLIT>
__global__ __launch_bounds__(WIDE_THREADS, 2) void gemm_fp8_block_tile_kernel(BlockArgs w) {
#ifdef __HIP_DEVICE_COMPILE__
  using S = WideShape<WM, TM, TN, NA, NB>;
  constexpr int WN = S::WN, BM = S::BM, BN = S::BN, PA = S::PA, PB = S::PB, LA = S::LA, LB = S::LB;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  lds_u8_t* const base = (lds_u8_t*)lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN, r16 = lane & 15, quad = lane >> 4;
  const int K = w.K, nk = (K + GROUP - 1) / GROUP, tail_chunks = (K % GROUP) / 16;

  // Chunk c of row r lies at c ^ key: a's bits 1, 2, 3 of r, b's bits 1, 3, 4.  MFMA row r of the pair of column tiles
  // (2 p, 2 p + 1) is column 32 p + 8 (r / 4) + 4 (tile & 1) + r % 4 of the wave's; a last single tile keeps the order.
  auto key_b = [](int row) { return (uint32_t)(((row >> 1) & 1) | ((row >> 3) & 3) << 1); };
  const int pair_row = wn * 16 * TN + (r16 >> 2) * 8 + (r16 & 3), single_row = wn * 16 * TN + 16 * (TN - 1) + r16;
  const lds_u8_t* const a0 = base + (wm * 16 * TM + r16) * ROWB + ((quad ^ (r16 >> 1)) << 4);
  const lds_u8_t* const a1 = base + (wm * 16 * TM + r16) * ROWB + (((4 + quad) ^ (r16 >> 1)) << 4);
  const lds_u8_t* const b0 = base + S::AT_B + pair_row * ROWB + ((quad ^ key_b(pair_row)) << 4);
  const lds_u8_t* const b1 = base + S::AT_B + pair_row * ROWB + (((4 + quad) ^ key_b(pair_row)) << 4);
  [[maybe_unused]] const lds_u8_t* const c0 = base + S::AT_B + single_row * ROWB + ((quad ^ key_b(single_row)) << 4);
  [[maybe_unused]] const lds_u8_t* const c1 = base + S::AT_B + single_row * ROWB + (((4 + quad) ^ key_b(single_row)) << 4);
  const lds_u8_t* const at_scale = base + S::AT_S + (wm * 16 * TM + r16) * 4;
  auto fragment_b = [&](int j, uint32_t use) {
    if (TN % 2 && j == TN - 1) return fragment(c0 + use, c1 + use);
    return fragment(b0 + use + (j >> 1) * 4096 + (j & 1) * 512, b1 + use + (j >> 1) * 4096 + (j & 1) * 512);
  };

  // Loads: wave w fills the 8-row blocks w, w + 8, ... of a panel.
  uint32_t va[LA], vb[LB];
  const int chunk_a = (lane & 7) ^ ((wave & 1) << 2 | lane >> 4), chunk_b = (lane & 7) ^ (((lane >> 4) & 1) | (wave & 3) << 1);
#pragma unroll
  for (int l = 0; l < LA; ++l) va[l] = (uint32_t)((wave + 8 * l) * 8 + (lane >> 3)) * (uint32_t)K + (chunk_a << 4);
#pragma unroll
  for (int l = 0; l < LB; ++l)
    vb[l] = (wave + 8 * l) * 8 < BN ? (uint32_t)((wave + 8 * l) * 8 + (lane >> 3)) * (uint32_t)K + (chunk_b << 4) : OUT_OF_RANGE;

  const uint32_t past_a = TAIL && chunk_a >= tail_chunks ? OUT_OF_RANGE : 0u;  // of the last slab
  const uint32_t past_b = TAIL && chunk_b >= tail_chunks ? OUT_OF_RANGE : 0u;

  const int whole = w.tiles_m * w.tiles_n, num_tiles = SPLIT ? whole * w.parts : whole;
  for (int t = blockIdx.x; t < num_tiles; t += gridDim.x) {
    int pid = t;
    const int per_xcd = num_tiles / 8;
    if (t < per_xcd * 8) pid = (t & 7) * per_xcd + (t >> 3);
    // the part's slabs: `slabs` of them from `from` on
    const int part_of = SPLIT ? pid / whole : 0, from = SPLIT ? part_of * w.per : 0, slabs = SPLIT ? min(w.per, nk - from) : nk;
    pid -= part_of * whole;
    const int sweep = 4 * w.tiles_n, group = pid / sweep, first = group * 4, in_group = min(w.tiles_m - first, 4);
    const int m0 = (first + pid % sweep % in_group) * BM, n0 = pid % sweep / in_group * BN;
    const int rows = min(w.M - m0, BM), cols = min(w.N - n0, BN);
    const __amdgpu_buffer_rsrc_t da = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(w.a) + (size_t)m0 * K, 0, (uint32_t)rows * (uint32_t)K, 0x00020000);
    const __amdgpu_buffer_rsrc_t db = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(w.b) + (size_t)n0 * K, 0, (uint32_t)cols * (uint32_t)K, 0x00020000);
    const float* const scales = w.a_scales + (int64_t)m0 * w.scale_row;
    const int scale_part = wave % (BM / 64) * 64;  // 64 rows' scales a wave, some of them twice: all waves count alike
    const uint32_t my_scale = (uint32_t)min(scale_part + lane, rows - 1) * (uint32_t)w.scale_row * 4u;
    // Past the last slab loads bring that one again and fragments are read that nobody uses: branches cost more (a
    // second set of registers for b's fragments, and spills).
    auto load_a = [&](int l, int slab, uint32_t at, uint32_t at_s) {
      const int k = from + min(slab, slabs - 1);
      if (l == LA) {
        load_scales(scales + k * w.scale_block, my_scale, base + S::AT_S + at_s + scale_part * 4);
        return;
      }
      const uint32_t off = TAIL ? va[l] | (k == nk - 1 ? past_a : 0u) : va[l];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(da, (lds_void_t*)(base + at + (wave + 8 * l) * 1024), 16, off,
                                               (uint32_t)k * ROWB, 0, 0);
    };
    auto load_b = [&](int l, int slab, uint32_t at) {
      const int k = from + min(slab, slabs - 1);
      const uint32_t off = TAIL ? vb[l] | (k == nk - 1 ? past_b : 0u) : vb[l];
      const uint32_t to = BN % 64 == 0 || (wave + 8 * l) * 8 < BN ? S::AT_B + at + (wave + 8 * l) * 1024 : S::AT_NONE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(db, (lds_void_t*)(base + to), 16, off, (uint32_t)k * ROWB, 0, 0);
    };
    auto all_a = [&](int slab) {
#pragma unroll
      for (int l = 0; l <= LA; ++l) load_a(l, slab, slab * PA, slab * BM * 4);
    };
    auto all_b = [&](int slab) {
#pragma unroll
      for (int l = 0; l < LB; ++l) load_b(l, slab, slab * PB);
    };
    // The weight's scales: the wave's columns touch two blocks at most (one if it has 32, 64 or 128 columns).  Lane l
    // keeps those of slab l of 64.
    constexpr bool TWO = GROUP % (16 * TN) != 0;
    const int col = n0 + wn * 16 * TN, most_block = (w.N - 1) / GROUP;
    const float* const sb = w.b_scales + (int64_t)min(col / GROUP, most_block) * nk + from;
    const int64_t second = TWO && col / GROUP + 1 <= most_block ? nk : 0;
    const int border = GROUP - col % GROUP;  // columns of the first block
    float sb0 = sb[min(lane, slabs - 1)], sb1 = sb[min(lane, slabs - 1) + second];

    f32x4_t acc[TM][TN], part[S::RING];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int x = 0; x < S::RING; ++x) part[x] = f32x4_t{0, 0, 0, 0};
    float first_scale = 0.0f, second_scale = 0.0f;  // of the row of tiles before
    auto add = [&](int x, float in_first, float in_second) {  // the results of a slab's instruction x
      const int i = x / TN, j = x % TN;
      // (an even count of column tiles: the border lies between two pairs)
      const int column = TN % 2 == 0 || j == TN - 1 ? 16 * j : (j >> 1) * 32 + quad * 8;
      const float scale = !TWO || column < border ? in_first : in_second;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = __fmaf_rn(part[x % S::RING][e], scale, acc[i][j][e]);
    };

    // as the loop would have left it
    all_a(0), all_b(0), all_a(1), all_b(1);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(S::PENDING) : "memory");
    uint32_t use_a = 0, use_b = 0, use_s = 0;           // of the slab at work
    uint32_t fill_a = (NA - 1) * PA, fill_s = (NA - 1) * BM * 4, fill_b = (NB - 1) * PB;
    // what a last row sends out
    constexpr int IN_LAST_ROW = (TN + S::SPACE_LATE - 1) / S::SPACE_LATE;
#pragma unroll
    for (int l = 0; l < S::LATE && l < IN_LAST_ROW; ++l) {
      if (l <= LA) load_a(l, NA - 1, fill_a, fill_s);
      else load_b(l - LA - 1, NB - 1, fill_b);
    }
    i32x8_t fa[2], fb[TN];
    fa[0] = fragment(a0, a1);
    float sa = *(lds_f32_t*)at_scale;
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = fragment_b(j, 0);
    for (int slab = 0; slab < slabs; ++slab) {
      if (slab && slab % 64 == 0) {
        sb0 = sb[min(slab + lane, slabs - 1)];
        sb1 = sb[min(slab + lane, slabs - 1) + second];
        asm volatile("" : "+v"(sb0), "+v"(sb1));  // waited for here: not in every slab, for all loads under way
      }
      const float s0 = lane_value(sb0, slab & 63), s1 = lane_value(sb1, slab & 63);
      const uint32_t next_a = after(use_a, PA, NA), next_b = after(use_b, PB, NB), next_s = after(use_s, BM * 4, NA);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const float mine0 = sa * s0, mine1 = sa * s1;
        if (i == TM - 1) {
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(S::PENDING) : "memory");
          fill_a = use_a, fill_s = use_s;
          if (!S::EARLY) fill_b = use_b;
        }
        if (S::EARLY && i == 1) {  // every wave has multiplied with all of its fragments of b
          asm volatile("s_barrier" ::: "memory");
          fill_b = use_b;
        }
        const uint32_t at = i + 1 < TM ? use_a + (i + 1) * 2048 : next_a;
        fa[(i + 1) & 1] = fragment(a0 + at, a1 + at);
        sa = *(lds_f32_t*)(at_scale + (i + 1 < TM ? use_s + (i + 1) * 64 : next_s));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          part[(i * TN + j) % S::RING] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa[i & 1], f32x4_t{}, 0, 0, 0, 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          if (i == TM - 1) fb[j] = fragment_b(j, next_b);
          const int late = (i + 1) % TM * TN + j, early = (i - 1) * TN + j;  // instructions since the barriers
          if (late % S::SPACE_LATE == 0 && late / S::SPACE_LATE < S::LATE) {
            const int l = late / S::SPACE_LATE, from = i == TM - 1 ? slab : slab - 1;
            if (l <= LA) load_a(l, from + NA, fill_a, fill_s);
            else load_b(l - LA - 1, from + NB, fill_b);
          }
          if (S::EARLY && early >= 0 && early % S::SPACE_EARLY == 0 && early / S::SPACE_EARLY < LB)
            load_b(early / S::SPACE_EARLY, slab + 2, fill_b);
          // of this row, or of the one before (for the first row: the slab before)
          if (j >= S::LAG) add(i * TN + j - S::LAG, mine0, mine1);
          else add((i * TN + j - S::LAG + S::TOTAL) % S::TOTAL, first_scale, second_scale);
          __builtin_amdgcn_sched_barrier(0);
        }
        first_scale = mine0, second_scale = mine1;
      }
      use_a = next_a, use_b = next_b, use_s = next_s;
    }
#pragma unroll
    for (int j = TN - S::LAG; j < TN; ++j) add((TM - 1) * TN + j, first_scale, second_scale);
    // a lane holds row r16 of each row of tiles, columns 8 quad + 0 .. 7 of a pair of column tiles
    const int m = wm * 16 * TM + r16, c0 = wn * 16 * TN;
    if constexpr (SPLIT) {
      const __amdgpu_buffer_rsrc_t ds = __builtin_amdgcn_make_buffer_rsrc(
          w.sums + ((size_t)part_of * w.M + m0) * w.N + n0, 0, (uint32_t)rows * (uint32_t)w.N * 4u, 0x00020000);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int c = c0 + (TN % 2 && j == TN - 1 ? 16 * j + quad * 4 : (j >> 1) * 32 + quad * 8 + (j & 1) * 4);
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, acc[i][j]), ds,
                                                 c < cols ? ((uint32_t)(m + 16 * i) * (uint32_t)w.N + c) * 4u : OUT_OF_RANGE, 0, 0);
        }
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the next tile's slabs go where this one's were
      continue;
    }
    auto four = [&](int i, int j) {
      return u32x2_t{pack_out(acc[i][j][0], acc[i][j][1], w.half_out), pack_out(acc[i][j][2], acc[i][j][3], w.half_out)};
    };
    with_store_form(w.form, [&](auto form) {
      uint16_t* const to = w.out + (size_t)(m0 + m) * w.ldc + n0;
      const __amdgpu_buffer_rsrc_t dc = __builtin_amdgcn_make_buffer_rsrc(
          w.out + (size_t)m0 * w.ldc + n0, 0, (uint32_t)rows * (uint32_t)w.ldc * 2u, 0x00020000);
      constexpr int AUX = form() == kWideThrough ? kStoreThrough : 0;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const uint32_t row = (uint32_t)(m + 16 * i) * (uint32_t)w.ldc * 2u;
#pragma unroll
        for (int j = 0; j + 1 < TN; j += 2) {
          const int c = c0 + j * 16 + quad * 8;
          const u32x2_t x = four(i, j), y = four(i, j + 1);
          if (form() != kNarrowStores) {
            __builtin_amdgcn_raw_buffer_store_b128(u32x4_t{x.x, x.y, y.x, y.y}, dc, c < cols ? row + 2 * c : OUT_OF_RANGE, 0, AUX);
          } else if (m + 16 * i < rows) {
            if (c < cols) *reinterpret_cast<u32x2_t*>(to + (size_t)(16 * i) * w.ldc + c) = x;
            if (c + 4 < cols) *reinterpret_cast<u32x2_t*>(to + (size_t)(16 * i) * w.ldc + c + 4) = y;
          }
        }
        if (TN % 2) {
          const int c = c0 + 16 * (TN - 1) + quad * 4;
          const u32x2_t x = four(i, TN - 1);
          if (form() != kNarrowStores)
            __builtin_amdgcn_raw_buffer_store_b64(x, dc, c < cols ? row + 2 * c : OUT_OF_RANGE, 0, 0);
          else if (m + 16 * i < rows && c < cols) *reinterpret_cast<u32x2_t*>(to + (size_t)(16 * i) * w.ldc + c) = x;
        }
      }
    });
    // The next tile's slabs go where this one's were: what is still on its way there has to arrive first, the stores
    // behind it need not.
    if (w.form == kNarrowStores) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(TM * ((TN + 1) / 2)) : "memory");
  }
#endif
}

template <int MT, int NT, int STAGES, int LA>
int launch_split(BlockArgs w, int max_cus, int cus, hipStream_t hs) {
  constexpr int LDS = split_lds(MT, NT, STAGES);
  static std::atomic<bool> ok[kMaxDevices];
  const auto kernel = gemm_fp8_block_split_kernel<MT, NT, STAGES, LA>;
  if (int rc = allow_lds("gemm_fp8_block_nt", reinterpret_cast<const void*>(kernel), ok, LDS)) return rc;
  // tiles just wide enough for a whole number of workgroups per compute unit
  w.tiles_m = (w.M + 8 * LA - 1) / (8 * LA);
  const int64_t full = (w.N + 32 * NT - 1) / (32 * NT), rounds = (w.tiles_m * full + cus - 1) / cus;
  const int64_t columns = std::max<int64_t>(full, cus * rounds / w.tiles_m);
  w.cols = (int)std::min<int64_t>(32 * NT, ((w.N + columns - 1) / columns + 3) / 4 * 4);
  w.tiles_n = (w.N + w.cols - 1) / w.cols;
  int64_t grid = (int64_t)w.tiles_m * w.tiles_n;
  if (max_cus > 0 && grid > max_cus) grid = max_cus;
  launch_kernel(kernel, dim3((unsigned)grid), dim3(SPLIT_THREADS), LDS, hs, w);
  return TW_OK;
}

template <int WM, int TM, int TN, int NA, int NB, bool SPLIT = false>
int launch_wide(BlockArgs w, int max_cus, int cus, hipStream_t hs) {
  using S = WideShape<WM, TM, TN, NA, NB>;
  static std::atomic<bool> ok[2][kMaxDevices];
  const bool tail = w.K % GROUP != 0;
  const auto kernel = tail ? gemm_fp8_block_tile_kernel<WM, TM, TN, NA, NB, true, SPLIT>
                           : gemm_fp8_block_tile_kernel<WM, TM, TN, NA, NB, false, SPLIT>;
  if (int rc = allow_lds("gemm_fp8_block_nt", reinterpret_cast<const void*>(kernel), ok[tail], S::LDS)) return rc;
  w.tiles_m = (w.M + S::BM - 1) / S::BM;
  w.tiles_n = (w.N + S::BN - 1) / S::BN;
  int64_t grid = (int64_t)w.tiles_m * w.tiles_n * (SPLIT ? w.parts : 1);
  // Through the L2 at once only where there is a tile a unit at most.  One: [1000, 3696] x [8192, 3696]^T 35.3 us, kept 37.5;
  // two, the loads of the second beside the stores of the first: [4096, 8192] x [7168, 8192]^T 228, kept 208.
  const int units = max_cus > 0 && max_cus < cus ? max_cus : cus;
  if (w.form == kWideThrough && grid > units) w.form = kWideStores;
  if (max_cus > 0 && grid > max_cus) grid = max_cus;
  launch_kernel(kernel, dim3((unsigned)grid), dim3(WIDE_THREADS), S::LDS, hs, w);
  return TW_OK;
}

// The tile shapes (WM, TM, TN, slabs of a and of b in LDS) with the time that a round of one tile a compute unit takes,
// relative to 256 x 224, measured at K = 8192 (106 us).  By area the large ones are alike (two rounds: 505 to 542 values
// a ns, 128 x 128 441), so what counts is how the tile count fits the units: [4096, 8192] x [7168, 8192] has 512 tiles of
// 256 x 224 and takes 205 us, with 192 x 256 256 us, 256 x 128 247, 128 x 128 292; [1000, 3696] x [8192, 3696] has 256
// tiles of 128 x 256: 38.6 us, with 256 x 224 54.5, 192 x 256 47.0, 128 x 128 47.8.  64 x 128: two of them fit a unit.
#define TW_WIDE_TILES(X)                                                                                    \
  X(4, 4, 7, 3, 2, 1.0) X(4, 4, 6, 3, 2, 0.87) X(2, 6, 4, 3, 2, 0.83) X(4, 4, 4, 3, 3, 0.61) X(2, 4, 4, 3, 3, 0.59) \
  X(2, 4, 2, 3, 3, 0.37) X(2, 2, 2, 3, 3, 0.22)

struct WideTile { int wm, tm, tn; double cost; };
#define TW_WIDE_TILE(WM, TM, TN, NA, NB, COST) {WM, TM, TN, COST},
constexpr WideTile kWideTiles[] = {TW_WIDE_TILES(TW_WIDE_TILE)};
#undef TW_WIDE_TILE

// The shape whose rounds take the least time; no shape changes a result bit (an element's slabs are added in order).
int launch_wide_for(const BlockArgs& w, int max_cus, int cus, hipStream_t hs) {
  const int units = max_cus > 0 && max_cus < cus ? max_cus : cus;
  const WideTile* best = &kWideTiles[0];
  double best_cost = 1e300;
  for (const WideTile& t : kWideTiles) {
    const int64_t bm = 16 * t.tm * t.wm, bn = 16 * t.tn * (8 / t.wm);
    const int64_t tiles = (w.M + bm - 1) / bm * ((w.N + bn - 1) / bn);
    const double cost = (double)((tiles + units - 1) / units) * t.cost;
    if (cost < best_cost) best = &t, best_cost = cost;
  }
#define TW_WIDE_LAUNCH(WM, TM, TN, NA, NB, COST) \
  if (best->wm == WM && best->tm == TM && best->tn == TN) return launch_wide<WM, TM, TN, NA, NB>(w, max_cus, cus, hs);
  TW_WIDE_TILES(TW_WIDE_LAUNCH)
#undef TW_WIDE_LAUNCH
  return set_error(TW_ERR_INVALID_ARGUMENT, "gemm_fp8_block_nt: no tile for %d rows", w.M);
}

// K divided: for more than 64 rows, where columns are few and tiles leave units idle or the inner dimension is long.  All
// times in us: a slab of a 256 x 224 tile 1.66 (the others as kWideTiles has them), 3 for a launch besides, 4 for the one that
// adds the sums, and those to memory and back; nothing reads b faster than memory gives it.  Undivided, up to 128 rows, a
// wave's slab takes 0.95, and this kernel gets a unit's lines at 50 GB/s beside a launch of 2.5 us.  [M, 8192] x [1024, 8192]^T, undivided / by this rule: 96 rows 18.7
// / 11.1, 200: 24.0 / 13.6, 512: 24.6 / 17.8, 1000: 25.0 / 20.9.  Left whole: [96, 8192] x [7168, 8192]^T (17.6; divided 16.3 and
// the launch that adds), [1000, 3696] x [8192, 3696]^T, [341, 2048] x [768, 2048]^T (8.7, of which the launch and the first slab 4).
constexpr double SPLIT_SLAB_US = 1.66, SPLIT_LAUNCH_US = 3.0, SPLIT_JOIN_US = 4.0, SPLIT_SUMS_A_US = 6e6, SPLIT_BYTES_A_US = 5e6,
                 SPLIT_SAVES_US = 1.5;
constexpr int64_t SPLIT_MAX_ROWS = 1024, SPLIT_MIN_SLABS = 2, SPLIT_MAX_N = 1 << 21;
// 64 x 128, 128 x 128 and 128 x 256 of kWideTiles
#define TW_BLOCK_SPLIT_TILES(X) X(2, 2, 2, 3, 3, 0.22) X(2, 4, 2, 3, 3, 0.37) X(2, 4, 4, 3, 3, 0.59)
struct BlockSplit { int tm, tn, parts, per; };

// The rows, N and K decide, no grid cap: the parts' sums differ in the order of the additions.
BlockSplit block_split(int64_t M, int64_t N, int64_t K, int cus) {
  const int64_t nk = (K + GROUP - 1) / GROUP;
  BlockSplit best = {0, 0, 1, (int)nk};
  if (M <= 64 || M > SPLIT_MAX_ROWS || N > SPLIT_MAX_N || nk < 2 * SPLIT_MIN_SLABS) return best;
  double least = 1e300;
  if (M > 128) {
    for (const WideTile& t : kWideTiles) {
      const int64_t bm = 16 * t.tm * t.wm, bn = 16 * t.tn * (8 / t.wm), tiles = (M + bm - 1) / bm * ((N + bn - 1) / bn);
      least = std::min(least, SPLIT_LAUNCH_US + SPLIT_SLAB_US * t.cost * (double)((tiles + cus - 1) / cus * nk));
    }
  } else {
    const int64_t rows = (M + 1) / 2, cols = std::min<int64_t>(64, (2 * N + cus - 1) / cus);
    least = 2.5 + std::max(0.95 * (double)((nk + 3) / 4), (double)((rows + cols) * K) / 50e3);
  }
  least -= SPLIT_SAVES_US;
  const double from_memory = (double)N * (double)K / SPLIT_BYTES_A_US;
#define TW_BLOCK_SPLIT_COST(WM, TM, TN, NA, NB, COST)                                                                   \
  {                                                                                                                    \
    const int64_t bm = 16 * TM * WM, bn = 16 * TN * (8 / WM), tiles = (M + bm - 1) / bm * ((N + bn - 1) / bn);         \
    for (int64_t parts = 2; parts * tiles <= cus && parts * SPLIT_MIN_SLABS <= nk; ++parts) {                          \
      const int64_t per = (nk + parts - 1) / parts;                                                                    \
      const double slabs = SPLIT_SLAB_US * COST * (double)per;                                                         \
      const double us = std::max(slabs, from_memory) + 0.1 * slabs + SPLIT_LAUNCH_US + SPLIT_JOIN_US +                 \
                        8.0 * (double)parts * (double)M * (double)N / SPLIT_SUMS_A_US;                                 \
      if (us < least) least = us, best = {TM, TN, (int)((nk + per - 1) / per), (int)per};                              \
    }                                                                                                                  \
  }
  TW_BLOCK_SPLIT_TILES(TW_BLOCK_SPLIT_COST)
#undef TW_BLOCK_SPLIT_COST
  return best;
}

constexpr int JOIN_THREADS = 256;
__global__ __launch_bounds__(JOIN_THREADS) void block_join_kernel(BlockArgs w) {
  const int across = w.N / 4;
  const int64_t step = (int64_t)gridDim.x * JOIN_THREADS, n = (int64_t)w.M * across;
  for (int64_t i = (int64_t)blockIdx.x * JOIN_THREADS + threadIdx.x; i < n; i += step) {
    const int64_t row = i / across;
    const int c = (int)(i - row * across) * 4;
    const float* p = w.sums + row * w.N + c;
    f32x4_t s = *reinterpret_cast<const f32x4_t*>(p);
#pragma unroll 4
    for (int x = 1; x < w.parts; ++x) {
      p += (int64_t)w.M * w.N;
      s += *reinterpret_cast<const f32x4_t*>(p);
    }
    *reinterpret_cast<uint2*>(w.out + row * w.ldc + c) = make_uint2(pack_out(s.x, s.y, w.half_out), pack_out(s.z, s.w, w.half_out));
  }
}

int launch_block_split(const char* what, BlockArgs w, const BlockSplit& split, float* sums, int max_cus, int cus, hipStream_t hs) {
  w.sums = sums, w.parts = split.parts, w.per = split.per;
  int rc = TW_OK;
#define TW_BLOCK_SPLIT_LAUNCH(WM, TM, TN, NA, NB, COST) \
  if (split.tm == TM && split.tn == TN) rc = launch_wide<WM, TM, TN, NA, NB, true>(w, max_cus, cus, hs);
  TW_BLOCK_SPLIT_TILES(TW_BLOCK_SPLIT_LAUNCH)
#undef TW_BLOCK_SPLIT_LAUNCH
  if (rc) return rc;
  if ((rc = finish_launch(what))) return rc;
  const int64_t groups = ((int64_t)w.M * (w.N / 4) + JOIN_THREADS - 1) / JOIN_THREADS;
  launch_kernel(block_join_kernel, capped_grid(groups, max_cus), dim3(JOIN_THREADS), 0, hs, w);
  return TW_OK;
}

}  // namespace

int run_quant_fp8_groups(void* out, float* scales, int64_t scale_row, int64_t scale_group, const void* input,
                         int64_t ld_in, int64_t M, int64_t K, int act, int dtype, void* stream) {
  const char* what = "quant_fp8_groups";
  if (M < 0 || K <= 0 || M > INT32_MAX - QUANT_ROWS || K > INT32_MAX / 4)  // (rows of a last group are counted past M)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: bad shape, %lld rows of %lld", what, (long long)M, (long long)K);
  if (act > TW_ACT_GELU_TANH) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, act);
  if (dtype != TW_DTYPE_BF16 && dtype != TW_DTYPE_F16 && dtype != TW_DTYPE_F32)
    return set_error(TW_ERR_DTYPE, "%s: unknown dtype %d", what, dtype);
  const int64_t width = act >= 0 ? 2 * K : K, size = dtype == TW_DTYPE_F32 ? 4 : 2;
  if (M > 1 && ld_in < width)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: rows of %lld at a stride of %lld", what, (long long)width,
                     (long long)ld_in);
  if (M == 0) return TW_OK;
  if (!out || !scales || !input) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  if (reinterpret_cast<uintptr_t>(input) % size || reinterpret_cast<uintptr_t>(scales) % 4)
    return set_error(TW_ERR_ALIGNMENT, "%s: input and scales must be aligned to their elements", what);
  QuantArgs w = {};
  w.out = static_cast<uint8_t*>(out);
  w.scales = scales;
  w.input = input;
  w.scale_row = scale_row, w.scale_group = scale_group, w.ld_in = ld_in;
  w.M = (int)M, w.K = (int)K, w.groups = (int)((K + GROUP - 1) / GROUP), w.act = act < 0 ? -1 : act;
  const int64_t grid = (M + QUANT_ROWS - 1) / QUANT_ROWS * w.groups;
  if (grid > INT32_MAX) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: too large", what);
  const bool vec = K % 8 == 0 && ld_in * size % 16 == 0 && reinterpret_cast<uintptr_t>(input) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 8 == 0;
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  if (dtype == TW_DTYPE_BF16) launch_quant<TW_DTYPE_BF16>(w, vec, grid, hs);
  else if (dtype == TW_DTYPE_F16) launch_quant<TW_DTYPE_F16>(w, vec, grid, hs);
  else launch_quant<TW_DTYPE_F32>(w, vec, grid, hs);
  return finish_launch(what);
}

int64_t gemm_fp8_block_workspace(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > BLOCK_MAX_K)
    return set_error(TW_ERR_INVALID_ARGUMENT, "gemm_fp8_block_nt_workspace: bad shape M=%lld N=%lld K=%lld", (long long)M,
                     (long long)N, (long long)K);
  const int cus = device_compute_units();
  const BlockSplit s = block_split(M, N, K, cus > 0 ? cus : 256);
  return s.parts > 1 ? 4 * s.parts * M * N : 0;
}

int run_gemm_fp8_block_nt(void* out, const void* a, const float* a_scales, int64_t scale_row, int64_t scale_block,
                          const void* b, const float* b_scales, int64_t M, int64_t N, int64_t K, int64_t ldc, int dtype,
                          int max_cus, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "gemm_fp8_block_nt";
  if (M == 1) scale_row = 0;  // a single row's has no meaning
  if (M < 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > BLOCK_MAX_K || ldc < N)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: bad shape M=%lld N=%lld K=%lld ldc=%lld", what, (long long)M,
                     (long long)N, (long long)K, (long long)ldc);
  if (scale_row < 0 || scale_block < 0 || scale_row > BLOCK_MAX_SCALE_ROW)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: the scales of two rows may be 0 to %lld elements apart, got %lld", what,
                     (long long)BLOCK_MAX_SCALE_ROW, (long long)scale_row);
  if (K % 16 != 0 || N % 4 != 0 || ldc % 4 != 0)
    return set_error(TW_ERR_ALIGNMENT, "%s: needs K %% 16 == 0, N %% 4 == 0, ldc %% 4 == 0", what);
  if (dtype != TW_DTYPE_BF16 && dtype != TW_DTYPE_F16)
    return set_error(TW_ERR_DTYPE, "%s: out must be bf16 or fp16, got dtype %d", what, dtype);
  if (M == 0) return TW_OK;
  if (!out || !a || !a_scales || !b || !b_scales)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  auto misaligned = [](const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; };
  if (misaligned(a, 16) || misaligned(b, 16) || misaligned(out, 8) || misaligned(a_scales, 4) || misaligned(b_scales, 4))
    return set_error(TW_ERR_ALIGNMENT, "%s: needs 16-byte aligned a and b, 8-byte aligned out, 4-byte aligned scales",
                     what);
  BlockArgs w = {};
  w.out = static_cast<uint16_t*>(out);
  w.a = static_cast<const uint8_t*>(a);
  w.b = static_cast<const uint8_t*>(b);
  w.a_scales = a_scales, w.b_scales = b_scales;
  w.scale_row = scale_row, w.scale_block = scale_block, w.ldc = ldc;
  w.M = (int)M, w.N = (int)N, w.K = (int)K, w.half_out = dtype == TW_DTYPE_F16;
  w.form = ldc > BLOCK_WIDE_LDC ? kNarrowStores : store_form(out, N, ldc);
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  int cus = device_compute_units(), rc;
  if (cus <= 0) cus = 256;
  const BlockSplit split = block_split(M, N, K, cus);
  if (split.parts > 1) {
    const int64_t need = 4 * split.parts * M * N;
    if (!workspace || workspace_bytes < need)
      return set_error(TW_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %lld bytes, got %lld", what, (long long)need,
                       (long long)(workspace ? workspace_bytes : 0));
    if (misaligned(workspace, 256)) return set_error(TW_ERR_ALIGNMENT, "%s: needs a 256-byte aligned workspace", what);
    rc = launch_block_split(what, w, split, static_cast<float*>(workspace), max_cus, cus, hs);
  } else if (M <= 8) rc = launch_split<1, 1, 3, 1>(w, max_cus, cus, hs);
  else if (M <= 16) rc = launch_split<1, 1, 3, 2>(w, max_cus, cus, hs);
  else if (M <= 32) rc = launch_split<1, 1, 3, 4>(w, max_cus, cus, hs);
  else if (M <= 64) rc = launch_split<2, 1, 2, 8>(w, max_cus, cus, hs);
  else if (M <= 80) rc = launch_split<2, 2, 2, 5>(w, max_cus, cus, hs);
  else if (M <= 96) rc = launch_split<2, 2, 2, 6>(w, max_cus, cus, hs);
  else if (M <= 128) rc = launch_split<2, 2, 2, 8>(w, max_cus, cus, hs);
  else rc = launch_wide_for(w, max_cus, cus, hs);
  return rc ? rc : finish_launch(what);
}

}  // namespace tw
