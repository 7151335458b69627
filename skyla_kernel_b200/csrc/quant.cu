// Rows in 8 bits (q8.cuh): quantised from bfloat16 or 32-bit values, from a root-mean-square norm, and back.
#include "q8.cuh"
using namespace skyla;
using namespace skyla::q8;
SKYLA_EXPORT_ERROR_MESSAGE()

namespace {

template <typename TI>
__global__ void quantize_kernel(const TI* __restrict__ x, int64_t ldx, int width, int8_t* __restrict__ q, int64_t ldq,
                                float* __restrict__ scale) {
  __shared__ unsigned scratch[32];
  allow_dependents();
  grid_dependency_wait();
  const int64_t r = blockIdx.x;
  const TI* xr = x + r * ldx;
  unsigned m = 0;
  for (int i = threadIdx.x; i < width; i += blockDim.x) m = max(m, abs_bits(to_float(xr[i])));
  m = block_max(m, scratch);
  const bool bad = m >= kInfBits;
  const Step s = step_of(bad ? 0u : m);
  for (int i = threadIdx.x; i < width; i += blockDim.x) q[r * ldq + i] = bad ? 0 : (int8_t)round_q(to_float(xr[i]), s);
  if (threadIdx.x == 0) scale[r] = bad ? kNan : s.most / kMost;
}

// x += residual (rounded to x's type: the norm is that of the sum as it is kept), then the norm's row in 8 bits.
// With t = x * w the norm is t * inv, inv = 1 / sqrt(mean(x^2) + eps) one number for the row, and 127 t inv / (A inv)
// = 127 t / A: the integers do not depend on inv, which goes into the scale alone.
template <typename TX, typename TR, bool ADD>
__global__ void rmsnorm_q8_kernel(TX* __restrict__ x, int64_t ldx, const TR* __restrict__ residual, int64_t ldr, int width,
                                  const float* __restrict__ w, float eps, int8_t* __restrict__ q, int64_t ldq,
                                  float* __restrict__ scale) {
  __shared__ unsigned scratch[32];
  __shared__ float fscratch[32];
  allow_dependents();
  grid_dependency_wait();
  const int64_t r = blockIdx.x;
  TX* xr = x + r * ldx;
  float ss = 0.f;
  unsigned m = 0;
  for (int i = threadIdx.x; i < width; i += blockDim.x) {
    float v = to_float(xr[i]);
    if (ADD) {
      const TX kept = from_float<TX>(v + to_float(residual[r * ldr + i]));
      xr[i] = kept;
      v = to_float(kept);
    }
    ss = fmaf(v, v, ss);
    m = max(m, abs_bits(v * w[i]));
  }
  m = block_max(m, scratch);
  ss = block_sum(ss, fscratch);
  const float inv = 1.0f / sqrtf(ss / (float)width + eps);
  const bool bad = m >= kInfBits || abs_bits(ss) >= kInfBits || abs_bits(inv) >= kInfBits;
  const Step s = step_of(bad ? 0u : m);
  for (int i = threadIdx.x; i < width; i += blockDim.x)
    q[r * ldq + i] = bad ? 0 : (int8_t)round_q(to_float(xr[i]) * w[i], s);
  if (threadIdx.x == 0) scale[r] = bad ? kNan : s.most * inv / kMost;
}

template <typename TO>
__global__ void dequantize_kernel(const int8_t* __restrict__ q, int64_t ldq, const float* __restrict__ scale, int width,
                                  TO* __restrict__ out, int64_t ldo) {
  allow_dependents();
  grid_dependency_wait();
  const int64_t r = blockIdx.x;
  const float s = scale[r];
  for (int i = threadIdx.x; i < width; i += blockDim.x) out[r * ldo + i] = from_float<TO>((float)q[r * ldq + i] * s);
}

int threads_for(int width) { return width >= 2048 ? 512 : (width >= 512 ? 256 : 128); }

int check_sizes(const char* what, int64_t n_rows, int width, int64_t ld_in, int64_t ld_out) {
  if (width <= 0) return fail(kBadArgument, "%s: rows of %d", what, width);
  if (n_rows > 0x7fffffffLL) return fail(kBadArgument, "%s: more than 2^31 - 1 rows", what);
  if (ld_out < width || ld_in < 0) return fail(kBadArgument, "%s: row strides do not fit rows of %d", what, width);
  return kOk;
}
}  // namespace

extern "C" int skyla_quantize_rows(const void* x, int x_dtype, int64_t ldx, int64_t n_rows, int width, void* q, int64_t ldq,
                                   float* scale, cudaStream_t stream) {
  if (n_rows <= 0) return kOk;
  if (int rc = check_sizes("quantize_rows", n_rows, width, ldx, ldq)) return rc;
  SKYLA_DISPATCH(x_dtype, TI, {
    launch_overlapped(quantize_kernel<TI>, dim3((unsigned)n_rows), dim3(threads_for(width)), 0, stream, (const TI*)x, ldx,
                      width, (int8_t*)q, ldq, scale);
  });
  return check_launch("quantize_rows");
}

extern "C" int skyla_rmsnorm_q8(void* x, int x_dtype, int64_t ldx, const void* residual, int r_dtype, int64_t ldr,
                                int64_t n_rows, int width, const float* weight, float eps, void* q, int64_t ldq, float* scale,
                                cudaStream_t stream) {
  if (n_rows <= 0) return kOk;
  if (int rc = check_sizes("rmsnorm_q8", n_rows, width, ldx, ldq)) return rc;
  if (!(eps >= 0.f)) return fail(kBadArgument, "rmsnorm_q8: eps must not be negative");
  const dim3 grid((unsigned)n_rows), block(threads_for(width));
  if (residual == nullptr) {
    SKYLA_DISPATCH(x_dtype, TX, {
      launch_overlapped(rmsnorm_q8_kernel<TX, float, false>, grid, block, 0, stream, (TX*)x, ldx, (const float*)nullptr,
                        (int64_t)0, width, weight, eps, (int8_t*)q, ldq, scale);
    });
  } else {
    SKYLA_DISPATCH(x_dtype, TX, SKYLA_DISPATCH(r_dtype, TR, {
      launch_overlapped(rmsnorm_q8_kernel<TX, TR, true>, grid, block, 0, stream, (TX*)x, ldx, (const TR*)residual, ldr, width,
                        weight, eps, (int8_t*)q, ldq, scale);
    }););
  }
  return check_launch("rmsnorm_q8");
}

extern "C" int skyla_dequantize_rows(const void* q, int64_t ldq, const float* scale, int64_t n_rows, int width, void* out,
                                     int out_dtype, int64_t ldo, cudaStream_t stream) {
  if (n_rows <= 0) return kOk;
  if (int rc = check_sizes("dequantize_rows", n_rows, width, ldq, ldo)) return rc;
  SKYLA_DISPATCH(out_dtype, TO, {
    launch_overlapped(dequantize_kernel<TO>, dim3((unsigned)n_rows), dim3(threads_for(width)), 0, stream, (const int8_t*)q, ldq,
                      scale, width, (TO*)out, ldo);
  });
  return check_launch("dequantize_rows");
}
