// The product of two sets of 8-bit rows by four-element integer dot products: any strides and alignments, any width.
//   acc[t, f] = sum_k x[t, k] w[f, k]    exact: at most 131,071 products of at most 2^14 fit 32 bits
//   v = acc * x_scale[t] * w_scale[f]    in 32-bit floating point, in this order
// It serves the operands that the tensor-core kernels (gemm_q8.cu) do not take, rows that do not begin on multiples
// of 16 bytes, and is their twin in the tests: the sums are exact, so the two agree bit for bit.  Tiles of 64 x 64 in shared
// memory, sixteen sums a thread; bound by the integer pipe: 2,048 tokens x 4,096 to 6,144 in 1.5 ms (69 TOP/s).
#include "q8.cuh"
using namespace skyla;
using skyla::q8::scaled;
using skyla::q8::silu_times;
SKYLA_EXPORT_ERROR_MESSAGE()

namespace {
enum Mode : int { kStore = 0, kAccumulate = 1, kGated = 2 };
constexpr int TM = 64, TN = 64, TK = 64;  // tokens, outputs and bytes of K of a block's tile
constexpr int kThreads = 256;             // 16 x 16, each with 4 x 4 outputs
constexpr int kMaxWidth = 131071;

struct Args {
  const int8_t* x; int64_t ldx; const float* x_scale;
  const int8_t* w; int64_t ldw; const float* w_scale;
  void* y; int64_t ldy;
  int m, n, k;
};

// TK bytes of `rows` rows, zeros beyond the matrix; rows of 17 words, so that a column's words lie in different banks
__device__ __forceinline__ void load_tile(uint32_t (*tile)[TK / 4 + 1], const int8_t* src, int64_t ld, int64_t row0, int64_t n_rows,
                                          int k0, int k) {
  for (int i = threadIdx.x; i < 64 * (TK / 4); i += kThreads) {
    const int r = i / (TK / 4), c = i % (TK / 4);
    uint32_t v = 0;
    if (row0 + r < n_rows) {
      const int8_t* p = src + (row0 + r) * ld + k0 + 4 * c;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (k0 + 4 * c + b < k) v |= (uint32_t)(uint8_t)p[b] << (8 * b);
    }
    tile[r][c] = v;
  }
}

template <int MODE, typename TY>
__global__ void __launch_bounds__(kThreads) linear_q8_plain_kernel(Args a) {
  __shared__ uint32_t xs[TM][TK / 4 + 1], ws[TN][TK / 4 + 1], us[MODE == kGated ? TN : 1][TK / 4 + 1];
  allow_dependents();
  grid_dependency_wait();
  const int64_t t0 = (int64_t)blockIdx.y * TM, f0 = (int64_t)blockIdx.x * TN;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  int acc[4][4] = {}, up[4][4] = {};
  for (int k0 = 0; k0 < a.k; k0 += TK) {
    load_tile(xs, a.x, a.ldx, t0, a.m, k0, a.k);
    load_tile(ws, a.w, a.ldw, f0, a.n, k0, a.k);
    if (MODE == kGated) load_tile(us, a.w + (int64_t)a.n * a.ldw, a.ldw, f0, a.n, k0, a.k);
    __syncthreads();
#pragma unroll 4
    for (int c = 0; c < TK / 4; ++c) {
      int xv[4], wv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { xv[i] = (int)xs[ty + 16 * i][c]; wv[i] = (int)ws[tx + 16 * i][c]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(xv[i], wv[j], acc[i][j]);
      if (MODE == kGated) {
#pragma unroll
        for (int j = 0; j < 4; ++j) wv[j] = (int)us[tx + 16 * j][c];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) up[i][j] = __dp4a(xv[i], wv[j], up[i][j]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + ty + 16 * i;
    if (t >= a.m) continue;
    const float sx = a.x_scale[t];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t f = f0 + tx + 16 * j;
      if (f >= a.n) continue;
      TY* y = (TY*)a.y + t * a.ldy + f;
      const float v = scaled(acc[i][j], sx, a.w_scale[f]);
      if (MODE == kGated) {
        *y = from_float<TY>(silu_times(v, scaled(up[i][j], sx, a.w_scale[a.n + f])));
      } else if (MODE == kAccumulate) {
        *y = from_float<TY>(__fadd_rn(to_float(*y), v));
      } else {
        *y = from_float<TY>(v);
      }
    }
  }
}
}  // namespace

// x [m, k] and w [n (2n gated: the gate rows, then the up rows), k] in 8 bits with any row strides, scales for each row;
// mode 0: y = v, 1: y += v (float32), 2: y = silu(v of the gate) * v of the up (bfloat16).
extern "C" int skyla_linear_q8_plain(const void* x, int64_t ldx, const float* x_scale, const void* w, int64_t ldw,
                                     const float* w_scale, int m, int n, int k, void* y, int y_dtype, int64_t ldy, int mode,
                                     cudaStream_t stream) {
  if (m <= 0 || n <= 0) return kOk;
  if (k <= 0 || k > kMaxWidth) return fail(kBadArgument, "linear_q8: K=%d is outside 1..%d", k, kMaxWidth);
  if (mode < kStore || mode > kGated) return fail(kBadArgument, "linear_q8: unknown mode %d", mode);
  if ((mode == kAccumulate && y_dtype != kF32) || (mode == kGated && y_dtype != kBF16))
    return fail(kBadArgument, "linear_q8: mode %d does not write dtype code %d", mode, y_dtype);
  const Args a{(const int8_t*)x, ldx, x_scale, (const int8_t*)w, ldw, w_scale, y, ldy, m, n, k};
  const dim3 grid((unsigned)((n + TN - 1) / TN), (unsigned)((m + TM - 1) / TM));
  if (grid.y > 65535) return fail(kBadArgument, "linear_q8: %d tokens exceed the grid", m);
  const dim3 block(kThreads);
  if (mode == kGated) launch_overlapped(linear_q8_plain_kernel<kGated, __nv_bfloat16>, grid, block, 0, stream, a);
  else if (mode == kAccumulate) launch_overlapped(linear_q8_plain_kernel<kAccumulate, float>, grid, block, 0, stream, a);
  else SKYLA_DISPATCH(y_dtype, TY, { launch_overlapped(linear_q8_plain_kernel<kStore, TY>, grid, block, 0, stream, a); });
  return check_launch("linear_q8");
}
