// Gradients of the gated product  h = act(G) * U,  G = a bg^T,  U = a bu^T  (b = [bg; bu], [2 I, K]):
//
//   dG = dh U act'(G),  dU = dh act(G),  D = [dG dU]  [M, 2 I]
//   da = D b            [M, K]
//   db = D^T a          [2 I, K]
//
// One launch computes D from dh, G and U and writes it as it is, for da, and turned, for db, by tiles of 64 x 64 through
// LDS; both products then are "NN" (tw_gemm.hip), with b and a as they lie in memory.  D is rounded to bf16 once, as the
// matrix cores take it, and G and U were when they were kept: against 64 bits da and db of bf16 operands are off by
// 0.29 % in the mean square, with neither rounding by 0.17 % (their own).
//
// 4096 rows, K = 8192, I = 3584, medians of 60: D and D^T 43 us (88 MB read, 117 written: 4.8 TB/s; one of them 30), da
// 347 and db 380 by themselves, 704 in the launch that they share; with b and a turned beforehand as well, for the "NT"
// kernel, 104, 326 and 357, in a workspace of 302 MB instead of 118.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "tw_activation.h"
#include "tw_common.h"

namespace tw {

namespace {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

constexpr int TURN = 64;          // rows and columns of a tile
constexpr int TURN_PITCH = 66;    // elements of a tile's row in LDS: columns are read without conflicts
constexpr int GRAD_THREADS = 256;
constexpr int TURN_ROWS = GRAD_THREADS / (TURN / 4), TURN_STEPS = TURN / TURN_ROWS;  // four channels a thread and step

constexpr int64_t GRAD_MAX_K = 1 << 21;  // what the products take

struct GradArgs {
  const uint16_t *grad, *both;
  uint16_t *d, *d_turned;  // null: not wanted
  int64_t ld_grad, ld_both, pitch, pitch_turned;
  int M, I, across, tiles, act;
};

__device__ __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

// to[c][m0 ..] = the tile's columns c, four rows at a time.
__device__ __forceinline__ void write_turned(const uint16_t* tile, uint16_t* to, int columns, int m0, int64_t pitch) {
  for (int g = threadIdx.x; g < TURN * TURN / 4; g += GRAD_THREADS) {
    const int c = g / (TURN / 4), m = (g % (TURN / 4)) * 4;
    if (c < columns && m0 + m < pitch) {
      const uint16_t* p = tile + m * TURN_PITCH + c;
      *reinterpret_cast<uint2*>(to + c * pitch + m0 + m) =
          make_uint2(p[0] | (uint32_t)p[TURN_PITCH] << 16, p[2 * TURN_PITCH] | (uint32_t)p[3 * TURN_PITCH] << 16);
    }
  }
}

__global__ __launch_bounds__(GRAD_THREADS) void gated_grad_kernel(GradArgs w) {
  __shared__ __attribute__((aligned(16))) uint16_t tiles[2][TURN * TURN_PITCH];
  const int m = threadIdx.x / (TURN / 4), c = threadIdx.x % (TURN / 4) * 4;
  for (int t = blockIdx.x; t < w.tiles; t += gridDim.x) {
    const int c0 = t % w.across * TURN, m0 = t / w.across * TURN;
    uint2 dh[TURN_STEPS], g2[TURN_STEPS], u2[TURN_STEPS];  // all under way before the first is used
#pragma unroll
    for (int i = 0; i < TURN_STEPS; ++i) {
      const int row = m0 + m + i * TURN_ROWS;
      dh[i] = g2[i] = u2[i] = make_uint2(0, 0);  // past the rows: zeros, which give zeros
      if (row < w.M && c0 + c < w.I) {
        const uint16_t* both = w.both + row * w.ld_both + c0 + c;
        dh[i] = *reinterpret_cast<const uint2*>(w.grad + row * w.ld_grad + c0 + c);
        g2[i] = *reinterpret_cast<const uint2*>(both);
        u2[i] = *reinterpret_cast<const uint2*>(both + w.I);
      }
    }
    with_activation(w.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < TURN_STEPS; ++i) {
        const int row = m0 + m + i * TURN_ROWS;
        const float h[4] = {low(dh[i].x), high(dh[i].x), low(dh[i].y), high(dh[i].y)};
        const float gate[4] = {low(g2[i].x), high(g2[i].x), low(g2[i].y), high(g2[i].y)};
        const float up[4] = {low(u2[i].x), high(u2[i].x), low(u2[i].y), high(u2[i].y)};
        float x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float f, df;
          activation_and_slope<act()>(gate[e], f, df);
          x[e] = h[e] * up[e] * df;
          y[e] = h[e] * f;
        }
        const uint2 dg = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
        const uint2 du = make_uint2(pack2(y[0], y[1]), pack2(y[2], y[3]));
        if (w.d && row < w.M && c0 + c < w.I) {
          uint16_t* d = w.d + row * w.pitch + c0 + c;
          *reinterpret_cast<uint2*>(d) = dg;
          *reinterpret_cast<uint2*>(d + w.I) = du;
        }
        if (w.d && row < w.M && c0 + TURN >= w.I && 2 * w.I + c < w.pitch)  // behind D's columns: zeros
          *reinterpret_cast<uint2*>(w.d + row * w.pitch + 2 * w.I + c) = make_uint2(0, 0);
        if (w.d_turned) {
          uint32_t* p = reinterpret_cast<uint32_t*>(tiles[0] + (m + i * TURN_ROWS) * TURN_PITCH + c);
          p[0] = dg.x, p[1] = dg.y;
          p = reinterpret_cast<uint32_t*>(tiles[1] + (m + i * TURN_ROWS) * TURN_PITCH + c);
          p[0] = du.x, p[1] = du.y;
        }
      }
    });
    if (!w.d_turned) continue;
    __syncthreads();
    write_turned(tiles[0], w.d_turned + c0 * w.pitch_turned, w.I - c0, m0, w.pitch_turned);
    write_turned(tiles[1], w.d_turned + (int64_t)(w.I + c0) * w.pitch_turned, w.I - c0, m0, w.pitch_turned);
    __syncthreads();  // the next tile's values go where these were
  }
}

__global__ __launch_bounds__(GRAD_THREADS) void fill_zero_kernel(uint2* to, int64_t n) {
  for (int64_t i = blockIdx.x * (int64_t)GRAD_THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * GRAD_THREADS)
    to[i] = make_uint2(0, 0);
}

// A row of D or D^T: whole slabs of the products, zeros behind the last value.
int64_t whole_slabs(int64_t n) { return (n + TURN - 1) / TURN * TURN; }

int check_shape(const char* what, int64_t M, int64_t I, int64_t K) {
  if (M < 0 || I <= 0 || K <= 0 || M > INT32_MAX - TURN || I > INT32_MAX / 2 || K > INT32_MAX)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: bad shape M=%lld I=%lld K=%lld", what, (long long)M, (long long)I,
                     (long long)K);
  if (K % 8 != 0 || I % 4 != 0) return set_error(TW_ERR_ALIGNMENT, "%s: needs K %% 8 == 0, I %% 4 == 0", what);
  return TW_OK;
}

}  // namespace

int64_t gated_backward_workspace(int64_t M, int64_t I, int64_t K, bool want_a, bool want_b) {
  if (int rc = check_shape("gated_gemm_bf16_nt_backward_workspace", M, I, K)) return rc;
  // D, D turned, and the partial sums of one product after the other
  const int64_t pitch = whole_slabs(2 * I), pitch_turned = whole_slabs(M);
  const int64_t of_a = want_a && M ? gemm_bf16_nn_workspace(M, K, pitch) : 0;
  const int64_t of_b = want_b && M ? gemm_bf16_nn_workspace(2 * I, K, pitch_turned) : 0;
  return 2 * ((want_a ? M * pitch : 0) + (want_b ? 2 * I * pitch_turned : 0)) + std::max(of_a, of_b);
}

int run_gated_gemm_bf16_nt_backward(void* grad_a, void* grad_b, const void* grad_out, int64_t ld_grad, const void* a,
                                    const void* b, const void* both, int64_t ld_both, int64_t M, int64_t I, int64_t K,
                                    int act, int max_cus, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "gated_gemm_bf16_nt_backward";
  if (int rc = check_shape(what, M, I, K)) return rc;
  if (act < TW_ACT_SILU || act > TW_ACT_GELU_TANH)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, act);
  if (K > GRAD_MAX_K || (grad_a && 2 * I > GRAD_MAX_K) || (grad_b && whole_slabs(M) > GRAD_MAX_K))
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: K, 2 I and, for grad_b, the rows may be %lld at most", what,
                     (long long)GRAD_MAX_K);
  if (ld_grad < I || ld_grad % 4 != 0 || ld_both < 2 * I || ld_both % 4 != 0)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: rows of grad_out and gate_up need strides of at least %lld and %lld, "
                     "multiples of 4", what, (long long)I, (long long)(2 * I));
  auto misaligned = [](const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; };
  if (misaligned(grad_a, 8) || misaligned(grad_b, 8) || misaligned(grad_out, 8) || misaligned(both, 8) ||
      misaligned(a, 16) || misaligned(b, 16) || misaligned(workspace, 256))
    return set_error(TW_ERR_ALIGNMENT, "%s: needs 16-byte aligned a and b, a 256-byte aligned workspace and 8-byte "
                     "aligned gradients and gate_up", what);
  const hipStream_t hs = static_cast<hipStream_t>(stream);
  if (M == 0) {  // a sum over no rows
    if (!grad_b) return TW_OK;
    const int64_t n = 2 * I * K / 4;
    launch_kernel(fill_zero_kernel, capped_grid(std::min<int64_t>(1024, (n + GRAD_THREADS - 1) / GRAD_THREADS), max_cus),
                  dim3(GRAD_THREADS), 0, hs, static_cast<uint2*>(grad_b), n);
    return finish_launch(what);
  }
  if (!grad_a && !grad_b) return TW_OK;
  if (!grad_out || !a || !b || !both) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  const int64_t need = gated_backward_workspace(M, I, K, grad_a, grad_b);
  if (!workspace || workspace_bytes < need)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %lld bytes, got %lld", what, (long long)need,
                     (long long)(workspace ? workspace_bytes : 0));
  uint16_t* ws = static_cast<uint16_t*>(workspace);
  GradArgs w = {};
  w.grad = static_cast<const uint16_t*>(grad_out);
  w.both = static_cast<const uint16_t*>(both);
  w.pitch = whole_slabs(2 * I), w.pitch_turned = whole_slabs(M);
  if (grad_a) w.d = ws, ws += M * w.pitch;
  if (grad_b) w.d_turned = ws, ws += 2 * I * w.pitch_turned;
  float* const sums = reinterpret_cast<float*>(ws);
  w.ld_grad = ld_grad, w.ld_both = ld_both;
  w.M = (int)M, w.I = (int)I, w.act = act;
  w.across = (int)((I + TURN - 1) / TURN);
  const int64_t grid = (M + TURN - 1) / TURN * w.across;
  if (grid > INT32_MAX / 2) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: too large", what);
  w.tiles = (int)grid;
  launch_kernel(gated_grad_kernel, capped_grid(grid, max_cus), dim3(GRAD_THREADS), 0, hs, w);
  if (int rc = finish_launch(what)) return rc;
  NnOperands products[2];
  int count = 0;
  if (grad_a) products[count++] = {grad_a, w.d, b, M, w.pitch, 2 * I};
  if (grad_b) products[count++] = {grad_b, w.d_turned, a, 2 * I, w.pitch_turned, M};
  return run_gemm_bf16_nn(products, count, K, max_cus, sums, stream);
}

}  // namespace tw
