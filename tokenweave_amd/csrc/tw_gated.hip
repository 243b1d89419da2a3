// Gradients of the gated product  h = act(G) * U,  G = a bg^T,  U = a bu^T  (b = [bg; bu], [2 I, K]):
//
//   dG = dh U act'(G),  dU = dh act(G),  D = [dG dU]  [M, 2 I]
//   da = D b            [M, K]
//   db = D^T a          [2 I, K]
//
// Both products run on the "NT" kernels of tw_gemm.hip, whose operands have the inner dimension
// contiguous: db wants D and a with their rows turned into columns, da wants b so.  One launch makes all
// of that: it computes D from dh, G and U and writes it as it is and turned, and turns a and b, all by
// tiles of 64 x 64 through LDS.  D is rounded to bf16 once, as the matrix cores take it.
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
constexpr int TURN_THREADS = 256;
constexpr int TURN_ROWS = TURN_THREADS / (TURN / 4), TURN_STEPS = TURN / TURN_ROWS;  // four channels a thread and step

struct GradArgs {
  const uint16_t *grad, *both, *a, *b;
  uint16_t *d, *d_turned, *a_turned, *b_turned;  // d and b_turned for da, the other two for db; null: not wanted
  int64_t M, I, K, ld_grad, ld_both, pitch;      // pitch: M rounded up to whole slabs, the rest zeros
  int act;
  int64_t grad_tiles, a_tiles, b_tiles;
};

__device__ __forceinline__ float low(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

// Columns [c0, c0 + 64) of `to`'s rows: to[c][m0 ..] = the tile's columns, four at a time.
__device__ __forceinline__ void write_turned(const uint16_t* tile, uint16_t* to, int64_t c0, int64_t columns, int64_t m0,
                                             int64_t pitch, int64_t rows) {
  for (int g = threadIdx.x; g < TURN * TURN / 4; g += TURN_THREADS) {
    const int c = g / (TURN / 4), m = (g % (TURN / 4)) * 4;
    if (c0 + c < columns && m0 + m < rows) {
      const uint16_t* p = tile + m * TURN_PITCH + c;
      *reinterpret_cast<uint2*>(to + (c0 + c) * pitch + m0 + m) =
          make_uint2(p[0] | (uint32_t)p[TURN_PITCH] << 16, p[2 * TURN_PITCH] | (uint32_t)p[3 * TURN_PITCH] << 16);
    }
  }
}

// from [rows, columns] -> to [columns, pitch]; rows up to the next whole tile are zeros where the pitch holds them.
__device__ __forceinline__ void turn(uint16_t* tile, const uint16_t* from, uint16_t* to, int64_t rows, int64_t columns,
                                     int64_t pitch, int64_t t) {
  const int64_t across = (columns + TURN - 1) / TURN, m0 = t / across * TURN, c0 = t % across * TURN;
  const int m = threadIdx.x / (TURN / 4), c = threadIdx.x % (TURN / 4) * 4;
  uint2 v[TURN_STEPS];  // all under way before the first is used
#pragma unroll
  for (int i = 0; i < TURN_STEPS; ++i) {
    const int64_t row = m0 + m + i * TURN_ROWS;
    v[i] = make_uint2(0, 0);
    if (row < rows && c0 + c < columns) v[i] = *reinterpret_cast<const uint2*>(from + row * columns + c0 + c);
  }
#pragma unroll
  for (int i = 0; i < TURN_STEPS; ++i) {
    uint32_t* p = reinterpret_cast<uint32_t*>(tile + (m + i * TURN_ROWS) * TURN_PITCH + c);
    p[0] = v[i].x;
    p[1] = v[i].y;
  }
  __syncthreads();
  write_turned(tile, to, c0, columns, m0, pitch, pitch);
}

__global__ __launch_bounds__(TURN_THREADS) void gated_grad_kernel(GradArgs w) {
  __shared__ __attribute__((aligned(16))) uint16_t tiles[2][TURN * TURN_PITCH];
  int64_t t = blockIdx.x;
  if (t >= w.grad_tiles) {
    t -= w.grad_tiles;
    if (t < w.a_tiles) turn(tiles[0], w.a, w.a_turned, w.M, w.K, w.pitch, t);
    else turn(tiles[0], w.b, w.b_turned, 2 * w.I, w.K, 2 * w.I, t - w.a_tiles);
    return;
  }
  const int64_t across = (w.I + TURN - 1) / TURN, m0 = t / across * TURN, c0 = t % across * TURN;
  const int m = threadIdx.x / (TURN / 4), c = threadIdx.x % (TURN / 4) * 4;
  uint2 dh[TURN_STEPS], g2[TURN_STEPS], u2[TURN_STEPS];
#pragma unroll
  for (int i = 0; i < TURN_STEPS; ++i) {
    const int64_t row = m0 + m + i * TURN_ROWS;
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
      const int64_t row = m0 + m + i * TURN_ROWS;
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
        uint16_t* d = w.d + row * 2 * w.I + c0 + c;
        *reinterpret_cast<uint2*>(d) = dg;
        *reinterpret_cast<uint2*>(d + w.I) = du;
      }
      if (w.d_turned) {
        uint32_t* p = reinterpret_cast<uint32_t*>(tiles[0] + (m + i * TURN_ROWS) * TURN_PITCH + c);
        p[0] = dg.x, p[1] = dg.y;
        p = reinterpret_cast<uint32_t*>(tiles[1] + (m + i * TURN_ROWS) * TURN_PITCH + c);
        p[0] = du.x, p[1] = du.y;
      }
    }
  });
  if (!w.d_turned) return;
  __syncthreads();
  write_turned(tiles[0], w.d_turned, c0, w.I, m0, w.pitch, w.pitch);
  write_turned(tiles[1], w.d_turned + w.I * w.pitch, c0, w.I, m0, w.pitch, w.pitch);
}

__global__ __launch_bounds__(TURN_THREADS) void fill_zero_kernel(uint2* to, int64_t n) {
  for (int64_t i = blockIdx.x * (int64_t)TURN_THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * TURN_THREADS)
    to[i] = make_uint2(0, 0);
}

int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// Places of the four buffers in the workspace, in elements; a 256-byte boundary each.
struct GradPlaces { int64_t d, b_turned, d_turned, a_turned, total; };
GradPlaces grad_places(int64_t M, int64_t I, int64_t K, bool want_a, bool want_b) {
  const int64_t pitch = up_to(M, TURN);
  GradPlaces p = {};
  auto take = [&](int64_t n) { const int64_t at = p.total; p.total += up_to(n, 128); return at; };
  if (want_a) p.d = take(M * 2 * I), p.b_turned = take(K * 2 * I);
  if (want_b) p.d_turned = take(2 * I * pitch), p.a_turned = take(K * pitch);
  return p;
}

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
  return M == 0 ? 0 : 2 * grad_places(M, I, K, want_a, want_b).total;
}

int run_gated_gemm_bf16_nt_backward(void* grad_a, void* grad_b, const void* grad_out, int64_t ld_grad, const void* a,
                                    const void* b, const void* both, int64_t ld_both, int64_t M, int64_t I, int64_t K,
                                    int act, int max_cus, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "gated_gemm_bf16_nt_backward";
  if (int rc = check_shape(what, M, I, K)) return rc;
  if (act < TW_ACT_SILU || act > TW_ACT_GELU_TANH)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", what, act);
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
    launch_kernel(fill_zero_kernel, dim3((unsigned)std::min<int64_t>(1024, (n + TURN_THREADS - 1) / TURN_THREADS)),
                  dim3(TURN_THREADS), 0, hs, static_cast<uint2*>(grad_b), n);
    return finish_launch(what);
  }
  if (!grad_a && !grad_b) return TW_OK;
  if (!grad_out || !a || !b || !both) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: null pointer argument", what);
  const GradPlaces p = grad_places(M, I, K, grad_a, grad_b);
  if (!workspace || workspace_bytes < 2 * p.total)
    return set_error(TW_ERR_INVALID_ARGUMENT, "%s: needs a workspace of %lld bytes, got %lld", what,
                     (long long)(2 * p.total), (long long)(workspace ? workspace_bytes : 0));
  uint16_t* ws = static_cast<uint16_t*>(workspace);
  GradArgs w = {};
  w.grad = static_cast<const uint16_t*>(grad_out);
  w.both = static_cast<const uint16_t*>(both);
  w.a = static_cast<const uint16_t*>(a);
  w.b = static_cast<const uint16_t*>(b);
  w.M = M, w.I = I, w.K = K, w.ld_grad = ld_grad, w.ld_both = ld_both, w.act = act;
  w.pitch = up_to(M, TURN);
  const int64_t row_tiles = w.pitch / TURN, k_tiles = up_to(K, TURN) / TURN;
  w.grad_tiles = row_tiles * (up_to(I, TURN) / TURN);
  if (grad_a) w.d = ws + p.d, w.b_turned = ws + p.b_turned, w.b_tiles = up_to(2 * I, TURN) / TURN * k_tiles;
  if (grad_b) w.d_turned = ws + p.d_turned, w.a_turned = ws + p.a_turned, w.a_tiles = row_tiles * k_tiles;
  const int64_t grid = w.grad_tiles + w.a_tiles + w.b_tiles;
  if (grid > INT32_MAX) return set_error(TW_ERR_INVALID_ARGUMENT, "%s: too large", what);
  launch_kernel(gated_grad_kernel, dim3((unsigned)grid), dim3(TURN_THREADS), 0, hs, w);
  if (int rc = finish_launch(what)) return rc;
  if (grad_a)
    if (int rc = run_gemm_bf16_nt(grad_a, w.d, w.b_turned, nullptr, M, K, 2 * I, K, max_cus, stream)) return rc;
  if (grad_b) return run_gemm_bf16_nt(grad_b, w.d_turned, w.a_turned, nullptr, 2 * I, K, w.pitch, K, max_cus, stream);
  return TW_OK;
}

}  // namespace tw
