// C ABI launcher of aitamd_quantize_rows: rows of fp16 / bf16 to 8-bit integers with one scale a row,
//     scale[r] = max_c |x[r, c]| / 127,   q[r, c] = the whole number nearest to 127 x[r, c] / max_c |x[r, c]|
// (ties to even).  127 x is exact in 32 bits, and the quotient of two such numbers of 11 significant bits is never so near to
// the middle between two whole numbers that its rounding to 32 bits decides: the integers are those of exact arithmetic.
// A multiplication by 127 / max instead of the division would not have that.
//
// Bound: memory, 2 bytes read and 1 written an element.  A row is held in registers between its maximum and its
// integers; only rows beyond 16384 columns are read a second time (from the caches, for the most part).
#include "../../include/aitemplate_amd_kernels.h"
#include "common.hpp"
#include "device.hpp"
#include "errors.hpp"

namespace aitamd {
namespace {

struct QuantizeParams {
  const void* x;
  int8_t* q;
  float* scale;
  int64_t rows, ldx, ldq;
  int32_t columns;
};

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

template <class T>
AITAMD_DEVICE float to_whole(uint16_t bits, float factor, float divisor) {
  // (the bits by value: a bit cast of a vector's element itself takes the vector's first)
  return __builtin_rintf(ElemTraits<T>::to_float(__builtin_bit_cast(T, bits)) * factor / divisor);
}

// the 8 elements at column c (those past the row as zeros)
template <class T>
AITAMD_DEVICE u16x8 row_piece(const T* x, int c, int columns) {
  u16x8 v = {};
  if (c + 8 <= columns) {
    v = load_vec<u16x8>(x + c);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < columns) v[j] = __builtin_bit_cast(uint16_t, x[c + j]);
  }
  return v;
}

// NT threads a row (16, 64: as many rows a workgroup as fit), HELD pieces of 8 elements a thread in registers; 0: rows of any length, read twice
template <class T, int NT, int HELD>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantizeParams p) {
  constexpr int ROWS = 256 / NT;
  constexpr uint32_t kInf = std::is_same_v<T, f16> ? 0x7c00u : 0x7f80u;
  __shared__ uint32_t of_wave[4];
  const int lane = threadIdx.x % NT;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / NT;
  if (ROWS > 1 && row >= p.rows) return;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.ldx;
  int8_t* q = p.q + row * p.ldq;
  u16x8 v[HELD > 0 ? HELD : 1];
  // The largest magnitude, as a whole number: its order is that of the bits without the sign, NaN on top of infinity.
  u16x8 most8 = {};
  auto take = [&](u16x8 w) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint16_t m = w[j] & 0x7fff;
      most8[j] = m > most8[j] ? m : most8[j];
    }
  };
  if constexpr (HELD > 0) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) v[i] = row_piece(x, (i * NT + lane) * 8, p.columns);
#pragma unroll
    for (int i = 0; i < HELD; ++i) take(v[i]);
  } else {
    for (int64_t c = lane * 8; c < p.columns; c += NT * 8) take(row_piece(x, (int)c, p.columns));
  }
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) bits = most8[j] > bits ? most8[j] : bits;
#pragma unroll
  for (int d = NT < 64 ? NT / 2 : 32; d > 0; d >>= 1) {
    const uint32_t other = __shfl_xor(bits, d);
    bits = other > bits ? other : bits;
  }
  if constexpr (NT == 256) {
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) bits = of_wave[w] > bits ? of_wave[w] : bits;
  }
  const float most = ElemTraits<T>::to_float(__builtin_bit_cast(T, (uint16_t)bits));
  // (a row with an infinity or a NaN has no scale: NaN, which makes every product with it one; a row of zeros has scale 0)
  if (lane == 0) p.scale[row] = bits >= kInf ? __builtin_nanf("") : most / 127.0f;
  const bool zeros = bits == 0 || bits >= kInf;
  // (127 times a bfloat16 may leave the range of 32 bits: both sides of the division 2^-32 times as large there)
  const float shrink = most > 0x1p100f ? 0x1p-32f : 1.0f, factor = 127.0f * shrink, divisor = most * shrink;
  auto put = [&](u16x8 w, int c) {
    u32x2 o = {};
    if (!zeros) {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j / 4] |= ((uint32_t)(int)to_whole<T>(w[j], factor, divisor) & 0xffu) << (8 * (j % 4));
    }
    if (c + 8 <= p.columns) {
      store_vec(q + c, o);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < p.columns) q[c + j] = (int8_t)(o[j / 4] >> (8 * (j % 4)));
    }
  };
  if constexpr (HELD > 0) {
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if ((i * NT + lane) * 8 < p.columns) put(v[i], (i * NT + lane) * 8);
  } else {
    for (int64_t c = lane * 8; c < p.columns; c += NT * 8) put(row_piece(x, (int)c, p.columns), (int)c);
  }
}

template <class T>
hipError_t launch_quantize(const QuantizeParams& p, hipStream_t stream) {
  // sixteen rows a workgroup where 16 lanes hold a row (200000 x 100: 73 us with a wave for each, 22 so), four where a wave does
  const auto kernel = p.columns <= 128 ? quantize_rows_kernel<T, 16, 1>
      : p.columns <= 512 ? quantize_rows_kernel<T, 64, 1>
      : p.columns <= 1024 ? quantize_rows_kernel<T, 64, 2>
      : p.columns <= 2048 ? quantize_rows_kernel<T, 256, 1>
      : p.columns <= 4096 ? quantize_rows_kernel<T, 256, 2>
      : p.columns <= 8192 ? quantize_rows_kernel<T, 256, 4>
      : p.columns <= 16384 ? quantize_rows_kernel<T, 256, 8>
                           : quantize_rows_kernel<T, 256, 0>;
  const int64_t rows_per_wg = p.columns <= 128 ? 16 : (p.columns <= 1024 ? 4 : 1);
  const int64_t most = most_workgroups(256) * rows_per_wg;
  for (int64_t row = 0; row < p.rows; row += most) {
    const QuantizeParams part{reinterpret_cast<const T*>(p.x) + row * p.ldx, p.q + row * p.ldq, p.scale + row,
                              p.rows - row < most ? p.rows - row : most, p.ldx, p.ldq, p.columns};
    hipLaunchKernelGGL(kernel, dim3((unsigned)((part.rows + rows_per_wg - 1) / rows_per_wg)), dim3(256), 0, stream, part);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace
}  // namespace aitamd

extern "C" int aitamd_quantize_rows(int dtype, const void* x, int8_t* q, float* scale, int64_t rows, int64_t columns, int64_t ldx,
                                    int64_t ldq, void* stream) {
  using namespace aitamd;
  const char* who = "aitamd_quantize_rows";
  if (dtype != AITAMD_F16 && dtype != AITAMD_BF16) return fail("%s: bad dtype %d", who, dtype);
  if (rows < 0 || columns < 0) return fail("%s: negative dimension", who);
  if (rows == 0) return 0;
  if (!scale || (columns > 0 && (!x || !q))) return fail("%s: null pointer", who);
  if (rows > 0x7fffffffll || columns > 0x7ffff000ll) return fail("%s: dimension too large", who);
  if (rows > 1 && (ldx < columns || ldq < columns)) return fail("%s: a row pitch (%lld, %lld) is smaller than the row (%lld)", who,
                                                                (long long)ldx, (long long)ldq, (long long)columns);
  const QuantizeParams p{x, q, scale, rows, ldx, ldq, (int32_t)columns};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = dtype == AITAMD_F16 ? launch_quantize<f16>(p, s) : launch_quantize<bf16>(p, s);
  if (e != hipSuccess) return fail("%s: launch failed: %s", who, hipGetErrorString(e));
  return 0;
}
