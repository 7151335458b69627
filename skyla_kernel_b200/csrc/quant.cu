// Rows in 8 bits (q8.cuh): quantised from bfloat16 or 32-bit values, from a root-mean-square norm, and back.
// All three are bound by the memory where there are many rows.  A row belongs to one group of threads (a warp for short rows,
// else a block), which reads it once, 16 bytes a thread and load, keeps it in registers while the group agrees on the row's
// largest value (one reduction), and writes its integers.  Elements beyond what the registers hold (kKeep loads a thread) are
// read again.
// Rows that do not begin on multiples of 16 bytes, or whose width leaves part of a load, go by two elements, or one.
// 24,576 x 4,096 quantised: 54 us of bfloat16 (5.6 TB/s), 79 of 32 bits (6.3 TB/s), read back 48 (6.3 TB/s); the norm of
// 8,192 x 4,096 with a bfloat16 residual 59 (6.3 TB/s); eight rows of 4,096 take 1.6, 1.6 and 2.4.
// A prompt's rows are between the two: 2,048 x 12,288 quantised of bfloat16 in 17.4 us, where the memory takes 11.5 and the
// instructions 9.6 (10.7 M of a warp, 64 % of the issue slots of an active SM).  At 64 registers five blocks of 192 threads
// fit an SM, so the rows are 2.8 rounds of blocks that load, meet and compute in step, and an SM is active 76 % of the time.
// The norm of 2,048 x 4,096 in 32 bits without a residual takes 11.9 us (3.5 TB/s), of 8,192 x 4,096 37.5 (4.5 TB/s).
#include <type_traits>

#include "q8.cuh"
using namespace skyla;
using namespace skyla::q8;
SKYLA_EXPORT_ERROR_MESSAGE()

namespace {

template <typename T> struct Type { typedef T type; };
template <int BYTES> struct Word;
template <> struct Word<1> { typedef uint8_t type; };
template <> struct Word<2> { typedef uint16_t type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<16> { typedef uint4 type; };

// E neighbouring elements, in loads and stores of at most 16 bytes
template <typename T, int E>
struct Pack {
  static constexpr int kBytes = E * (int)sizeof(T), kPiece = kBytes < 16 ? kBytes : 16, kPieces = kBytes / kPiece;
  typedef typename Word<kPiece>::type W;
  union { W w[kPieces]; uint16_t h[kBytes / 2 > 0 ? kBytes / 2 : 1]; uint32_t u[kBytes / 4 > 0 ? kBytes / 4 : 1]; };
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) w[i] = reinterpret_cast<const W*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) reinterpret_cast<W*>(p)[i] = w[i];
  }
  __device__ __forceinline__ float get(int i) const {
    if (sizeof(T) == 4) return __uint_as_float(u[i]);
    return __uint_as_float((uint32_t)h[i] << 16);  // a bfloat16 is the upper half of a 32-bit value
  }
  // the largest of `most` and the elements' magnitudes, as bits of 32-bit values.  (Two 16-bit elements at a time.)
  __device__ __forceinline__ unsigned largest(unsigned most) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < E; ++i) most = max(most, u[i] & 0x7fffffffu);
      return most;
    } else if constexpr (E == 1) {
      return max(most, (unsigned)(h[0] & 0x7fffu) << 16);
    } else {
      unsigned two = 0;
#pragma unroll
      for (int i = 0; i < E / 2; ++i) two = __vmaxu2(two, u[i] & 0x7fff7fffu);
      return max(most, max(two << 16, two & 0xffff0000u));
    }
  }
  __device__ __forceinline__ void set(int i, float v) {
    if (sizeof(T) == 4) u[i] = __float_as_uint(v);
    else h[i] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
};

template <int E>
__device__ __forceinline__ void store_q(int8_t* p, const uint32_t* n) {
  if constexpr (E == 1) *p = (int8_t)n[0];
  else if constexpr (E == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)__byte_perm(n[0], n[1], 0x0040);
  else if constexpr (E == 4) *reinterpret_cast<uint32_t*>(p) = low_bytes(n);
  else *reinterpret_cast<uint2*>(p) = make_uint2(low_bytes(n), low_bytes(n + 4));
}

__device__ __constant__ uint32_t kZeros[16] = {};

// The threads of a row: `BLOCK` a block's, else a warp's
template <bool BLOCK>
struct Group {
  int64_t row; int rank, size;
  __device__ __forceinline__ Group() {
    if (BLOCK) { row = blockIdx.x; rank = threadIdx.x; size = blockDim.x; }
    else { row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); rank = threadIdx.x & 31; size = 32; }
  }
  // largest of the group's words and sum of its values, both with one meeting; the sum's order is fixed by the group
  __device__ __forceinline__ void meet(unsigned& most, float* sum) const {
    __shared__ unsigned tops[32];
    __shared__ float sums[32];
    most = __reduce_max_sync(0xffffffffu, most);
    if (sum != nullptr) *sum = warp_sum(*sum);
    if (!BLOCK) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
    if (lane == 0) {
      tops[warp] = most;
      if (sum != nullptr) sums[warp] = *sum;
    }
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, lane < n_warps ? tops[lane] : 0u);
    if (sum != nullptr) *sum = warp_sum(lane < n_warps ? sums[lane] : 0.f);
  }
};

template <typename T, int E, int kKeep, bool BLOCK, bool LONG>
__global__ void __launch_bounds__(kKeep == 8 ? 512 : 1024) quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t n_rows,
                                                                           int width, int8_t* __restrict__ q, int64_t ldq,
                                                                           float* __restrict__ scale) {
  allow_dependents();
  grid_dependency_wait();
  const Group<BLOCK> g;
  if (g.row >= n_rows) return;  // (whole warps: a block has one row only)
  const T* xr = x + g.row * ldx;
  int8_t* qr = q + g.row * ldq;
  const int first = g.rank * E, step = g.size * E;
  // kKeep loads of a thread from element e on, all in flight together
  auto load = [&](int e, Pack<T, E>* p) {
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
      if (e + j * step < width) p[j].load(xr + e + j * step);
  };
  unsigned most = 0;
  auto look = [&](int e, const Pack<T, E>* p) {
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
      if (e + j * step < width) most = p[j].largest(most);
  };
  Pack<T, E> kept[kKeep];
  load(first, kept);
  look(first, kept);
#pragma unroll 1
  for (int e = first + kKeep * step; LONG && e < width; e += kKeep * step) {
    Pack<T, E> more[kKeep];
    load(e, more);
    look(e, more);
  }
  g.meet(most, nullptr);
  if (most >= kInfBits) {  // the same for the whole group
    for (int e = first; e < width; e += step) store_q<E>(qr + e, kZeros);
    if (g.rank == 0) scale[g.row] = kNan;
    return;
  }
  const Step s = step_of(most);
  auto put = [&](int e, const Pack<T, E>* p) {
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
      if (e + j * step < width) {
        float v[E];
        uint32_t n[E];
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = p[j].get(i);
        round_q<E, sizeof(T) == 2>(v, s, n);
        store_q<E>(qr + e + j * step, n);
      }
  };
  put(first, kept);
#pragma unroll 1
  for (int e = first + kKeep * step; LONG && e < width; e += kKeep * step) {
    Pack<T, E> more[kKeep];
    load(e, more);
    put(e, more);
  }
  if (g.rank == 0) scale[g.row] = s.most / kMost;
}

// x += residual (rounded to x's type: the norm is that of the sum as it is kept), then the norm's row in 8 bits.
// With t = x * w the norm is t * inv, inv = 1 / sqrt(mean(x^2) + eps) one number for the row, and 127 t inv / (A inv)
// = 127 t / A: the integers do not depend on inv, which goes into the scale alone, so the sum of squares and the largest
// t are found in one pass and one meeting.
template <typename TX, typename TR, bool ADD, int E, int kKeep, bool BLOCK, bool LONG>
__global__ void __launch_bounds__(kKeep == 1 ? 1024 : 768) rmsnorm_q8_kernel(TX* __restrict__ x, int64_t ldx, const TR* __restrict__ residual, int64_t ldr, int64_t n_rows,
                                  int width, const float* __restrict__ w, float eps, int8_t* __restrict__ q, int64_t ldq,
                                  float* __restrict__ scale) {
  allow_dependents();
  grid_dependency_wait();
  const Group<BLOCK> g;
  if (g.row >= n_rows) return;
  TX* xr = x + g.row * ldx;
  const TR* rr = ADD ? residual + g.row * ldr : nullptr;
  int8_t* qr = q + g.row * ldq;
  const int first = g.rank * E, step = g.size * E;
  float ss = 0.f;
  unsigned most = 0;
  // kKeep loads of a thread from element e on, all in flight together: the sums written back, and their t
  auto take = [&](int e, float (*t)[E]) {
    Pack<TX, E> p[kKeep];
    Pack<TR, E> add[ADD ? kKeep : 1];
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
      if (e + j * step < width) {
        p[j].load(xr + e + j * step);
        if (ADD) add[j].load(rr + e + j * step);
      }
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
      if (e + j * step < width) {
        Pack<float, E> weight;
        weight.load(w + e + j * step);
        if (ADD) {
#pragma unroll
          for (int i = 0; i < E; ++i) p[j].set(i, p[j].get(i) + add[ADD ? j : 0].get(i));
          p[j].store(xr + e + j * step);
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float v = p[j].get(i);
          ss = fmaf(v, v, ss);
          t[j][i] = v * weight.get(i);
          most = max(most, abs_bits(t[j][i]));
        }
      }
  };
  float kept[kKeep][E];
  take(first, kept);
#pragma unroll 1
  for (int e = first + kKeep * step; LONG && e < width; e += kKeep * step) {
    float more[kKeep][E];
    take(e, more);
  }
  g.meet(most, &ss);
  // the same for the whole group (the mean square and eps may both be zero; the scale is one thread's work)
  if (most >= kInfBits || abs_bits(ss) >= kInfBits || (eps == 0.f && ss / (float)width == 0.f)) {
    for (int e = first; e < width; e += step) store_q<E>(qr + e, kZeros);
    if (g.rank == 0) scale[g.row] = kNan;
    return;
  }
  const Step s = step_of(most);
  auto put = [&](int e, const float* t) {
    uint32_t n[E];
    round_q<E, false>(t, s, n);
    store_q<E>(qr + e, n);
  };
#pragma unroll
  for (int j = 0; j < kKeep; ++j)
    if (first + j * step < width) put(first + j * step, kept[j]);
#pragma unroll 1
  for (int e = first + kKeep * step; LONG && e < width; e += kKeep * step) {  // (this thread wrote these sums itself)
    Pack<TX, E> p[kKeep];
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
      if (e + j * step < width) p[j].load(xr + e + j * step);
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
      if (e + j * step < width) {
        Pack<float, E> weight;
        weight.load(w + e + j * step);
        float t[E];
#pragma unroll
        for (int i = 0; i < E; ++i) t[i] = p[j].get(i) * weight.get(i);
        put(e + j * step, t);
      }
  }
  if (g.rank == 0) scale[g.row] = s.most * (1.0f / sqrtf(ss / (float)width + eps)) / kMost;
}

template <typename T, int E, bool BLOCK>
__global__ void __launch_bounds__(1024) dequantize_kernel(const int8_t* __restrict__ q, int64_t ldq, const float* __restrict__ scale, int64_t n_rows,
                                  int width, T* __restrict__ out, int64_t ldo) {
  allow_dependents();
  grid_dependency_wait();
  const Group<BLOCK> g;
  if (g.row >= n_rows) return;
  const int8_t* qr = q + g.row * ldq;
  T* o = out + g.row * ldo;
  const float s = scale[g.row];
  auto put = [&](int64_t e, const typename Word<E>::type& raw) {
    const int8_t* n = reinterpret_cast<const int8_t*>(&raw);
    Pack<T, E> p;
#pragma unroll
    for (int i = 0; i < E; ++i) p.set(i, (float)n[i] * s);
    p.store(o + e);
  };
  int64_t e = (int64_t)g.rank * E;
  const int64_t step = (int64_t)g.size * E;
  for (; e + 3 * step < width; e += 4 * step) {  // four loads in flight
    typename Word<E>::type raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j] = *reinterpret_cast<const typename Word<E>::type*>(qr + e + j * step);
#pragma unroll
    for (int j = 0; j < 4; ++j) put(e + j * step, raw[j]);
  }
  for (; e < width; e += step) put(e, *reinterpret_cast<const typename Word<E>::type*>(qr + e));
}

int check_sizes(const char* what, int64_t n_rows, int width, int64_t ld_in, int64_t ld_out) {
  if (width <= 0) return fail(kBadArgument, "%s: rows of %d", what, width);
  if (n_rows > 0x7fffffffLL) return fail(kBadArgument, "%s: more than 2^31 - 1 rows", what);
  if (ld_out < 0 || ld_in < 0) return fail(kBadArgument, "%s: row strides do not fit rows of %d", what, width);
  return kOk;
}
// Rows of `size`-byte elements that begin on multiples of `bytes`
bool rows_on(const void* p, int64_t ld, int size, int bytes) { return (uintptr_t)p % bytes == 0 && ld * size % bytes == 0; }

// How a row is shared out: threads, and loads that each keeps.  Four loads a thread where there are many rows: what a thread
// does once for its row, some 200 instructions, counts for that many, and more registers a thread cost more than that gives
// (norm of 8,192 x 4,096 with its residual: 74 / 59 / 80 us at two / four / eight loads).  The quantisation (`most_kept` 8),
// whose loads stay as they come, gains by eight for long rows and for many of bfloat16 (2,048 x 12,288: 20.7 to 17.1 us of
// bfloat16, 35 to 27 of 32 bits; 24,576 x 4,096 of bfloat16: 58.3 to 53.6; but 2,048 x 4,096: 7.3 to 8.4).
struct Shape { int threads; int keep; bool block; bool longer; };
Shape shape_for(int64_t n_rows, int width, int E, int most_kept) {
  const int64_t loads = ((int64_t)width + E - 1) / E;
  // a warp a row, eight rows a block
  if (loads <= 32 * 4 && n_rows >= 8) return {256, loads <= 32 ? 1 : 4, false, false};
  int64_t threads;
  if (n_rows < 592) {  // fewer than four blocks for each of 148 SMs: as many threads as loads, for the shortest way from the row's first byte to its last
    threads = loads <= 1024 ? loads : 512;
  } else {
    const bool eight = loads > 2048 || (E == 8 && (loads >= 1024 || n_rows >= 8192));
    threads = (loads + (eight ? most_kept : 4) - 1) / (eight ? most_kept : 4);
    if (threads > 512) threads = most_kept == 4 && loads <= 4 * 768 ? 768 : 512;
  }
  threads = threads < 64 ? 64 : (threads + 31) / 32 * 32;
  return {(int)threads, loads <= threads ? 1 : loads <= 4 * threads ? 4 : most_kept, true, loads > most_kept * threads};
}
dim3 grid_for(int64_t n_rows, const Shape& s) { return dim3((unsigned)(s.block ? n_rows : (n_rows + s.threads / 32 - 1) / (s.threads / 32))); }

template <typename T, int E>
void launch_quantize(const Shape& s, const void* x, int64_t ldx, int64_t n_rows, int width, void* q, int64_t ldq, float* scale,
                     cudaStream_t stream) {
  auto go = [&](auto kernel) {
    launch_overlapped(kernel, grid_for(n_rows, s), dim3(s.threads), 0, stream, (const T*)x, ldx, n_rows, width, (int8_t*)q, ldq, scale);
  };
  if (!s.block) s.keep == 1 ? go(quantize_kernel<T, E, 1, false, false>) : go(quantize_kernel<T, E, 4, false, false>);
  else if (s.longer) go(quantize_kernel<T, E, 8, true, true>);
  else s.keep == 1 ? go(quantize_kernel<T, E, 1, true, false>) : s.keep == 4 ? go(quantize_kernel<T, E, 4, true, false>) : go(quantize_kernel<T, E, 8, true, false>);
}
template <typename TX, typename TR, bool ADD, int E>
void launch_norm(const Shape& s, void* x, int64_t ldx, const void* residual, int64_t ldr, int64_t n_rows, int width, const float* w,
                 float eps, void* q, int64_t ldq, float* scale, cudaStream_t stream) {
  auto go = [&](auto kernel) {
    launch_overlapped(kernel, grid_for(n_rows, s), dim3(s.threads), 0, stream, (TX*)x, ldx, (const TR*)residual, ldr, n_rows, width,
                      w, eps, (int8_t*)q, ldq, scale);
  };
  if (!s.block) s.keep == 1 ? go(rmsnorm_q8_kernel<TX, TR, ADD, E, 1, false, false>) : go(rmsnorm_q8_kernel<TX, TR, ADD, E, 4, false, false>);
  else if (s.longer) go(rmsnorm_q8_kernel<TX, TR, ADD, E, 4, true, true>);
  else s.keep == 1 ? go(rmsnorm_q8_kernel<TX, TR, ADD, E, 1, true, false>) : go(rmsnorm_q8_kernel<TX, TR, ADD, E, 4, true, false>);
}
}  // namespace

extern "C" int skyla_quantize_rows(const void* x, int x_dtype, int64_t ldx, int64_t n_rows, int width, void* q, int64_t ldq,
                                   float* scale, cudaStream_t stream) {
  if (n_rows <= 0) return kOk;
  if (int rc = check_sizes("quantize_rows", n_rows, width, ldx, ldq)) return rc;
  SKYLA_DISPATCH(x_dtype, T, {
    constexpr int E = 16 / sizeof(T);
    if (width % E == 0 && rows_on(x, ldx, sizeof(T), 16) && rows_on(q, ldq, 1, E))
      launch_quantize<T, E>(shape_for(n_rows, width, E, 8), x, ldx, n_rows, width, q, ldq, scale, stream);
    else if (width % 2 == 0 && rows_on(x, ldx, sizeof(T), 2 * sizeof(T)) && rows_on(q, ldq, 1, 2))
      launch_quantize<T, 2>(shape_for(n_rows, width, 2, 8), x, ldx, n_rows, width, q, ldq, scale, stream);
    else
      launch_quantize<T, 1>(shape_for(n_rows, width, 1, 8), x, ldx, n_rows, width, q, ldq, scale, stream);
  });
  return check_launch("quantize_rows");
}

extern "C" int skyla_rmsnorm_q8(void* x, int x_dtype, int64_t ldx, const void* residual, int r_dtype, int64_t ldr,
                                int64_t n_rows, int width, const float* weight, float eps, void* q, int64_t ldq, float* scale,
                                cudaStream_t stream) {
  if (n_rows <= 0) return kOk;
  if (int rc = check_sizes("rmsnorm_q8", n_rows, width, ldx, ldq)) return rc;
  if (!(eps >= 0.f)) return fail(kBadArgument, "rmsnorm_q8: eps must not be negative");
  SKYLA_DISPATCH(x_dtype, TX, {
    // whether rows can go by e elements: x, residual, weight and q begin on as many whole ones (a load takes at most 16 bytes)
    auto on = [&](int e) {
      const int r_bytes = e * (r_dtype == kF32 ? 4 : 2), w_bytes = 4 * e;
      return width % e == 0 && rows_on(x, ldx, sizeof(TX), e * (int)sizeof(TX)) && rows_on(q, ldq, 1, e) &&
             (uintptr_t)weight % (w_bytes < 16 ? w_bytes : 16) == 0 &&
             (residual == nullptr || rows_on(residual, ldr, r_dtype == kF32 ? 4 : 2, r_bytes < 16 ? r_bytes : 16));
    };
    auto by = [&](auto e, auto tr, auto add) {
      constexpr int E = decltype(e)::value;
      launch_norm<TX, typename decltype(tr)::type, decltype(add)::value, E>(shape_for(n_rows, width, E, 4), x, ldx, residual, ldr, n_rows,
                                                                           width, weight, eps, q, ldq, scale, stream);
    };
    auto with = [&](auto tr, auto add) {
      // (four elements of a bfloat16 row with a 32-bit residual, for the registers' sake)
      constexpr int E = 16 / (decltype(add)::value && sizeof(typename decltype(tr)::type) > sizeof(TX) ? 4 : sizeof(TX));
      if (on(E)) by(std::integral_constant<int, E>(), tr, add);
      else if (on(2)) by(std::integral_constant<int, 2>(), tr, add);
      else by(std::integral_constant<int, 1>(), tr, add);
    };
    if (residual == nullptr) with(Type<float>(), std::false_type());
    else SKYLA_DISPATCH(r_dtype, TR, { with(Type<TR>(), std::true_type()); });
  });
  return check_launch("rmsnorm_q8");
}

extern "C" int skyla_dequantize_rows(const void* q, int64_t ldq, const float* scale, int64_t n_rows, int width, void* out,
                                     int out_dtype, int64_t ldo, cudaStream_t stream) {
  if (n_rows <= 0) return kOk;
  if (int rc = check_sizes("dequantize_rows", n_rows, width, ldq, ldo)) return rc;
  SKYLA_DISPATCH(out_dtype, T, {
    auto go = [&](auto kernel, const Shape& s) {
      launch_overlapped(kernel, grid_for(n_rows, s), dim3(s.threads), 0, stream, (const int8_t*)q, ldq, scale, n_rows, width, (T*)out, ldo);
    };
    const bool vec = width % 8 == 0 && rows_on(q, ldq, 1, 8) && rows_on(out, ldo, sizeof(T), 16);
    const bool two = !vec && width % 2 == 0 && rows_on(q, ldq, 1, 2) && rows_on(out, ldo, sizeof(T), 2 * sizeof(T));
    const Shape s = shape_for(n_rows, width, vec ? 8 : two ? 2 : 1, 4);
    if (vec) s.block ? go(dequantize_kernel<T, 8, true>, s) : go(dequantize_kernel<T, 8, false>, s);
    else if (two) s.block ? go(dequantize_kernel<T, 2, true>, s) : go(dequantize_kernel<T, 2, false>, s);
    else s.block ? go(dequantize_kernel<T, 1, true>, s) : go(dequantize_kernel<T, 1, false>, s);
  });
  return check_launch("dequantize_rows");
}
