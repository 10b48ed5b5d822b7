// Inverted dropout whose mask is never stored: y = keep ? x * scale : 0 [+ residual].
//
// keep(row, col) comes from one Philox-4x32-10 block for eight neighbouring
// columns of a row: counter {col / 8, row, offset lo, offset hi}, key = seed; its
// four words give 16 bits to each column (low half first), and the element stays
// when they are >= `cut` = round(p * 65536). scale = 65536 / (65536 - cut), so
// the expectation is exact for the probability that is really drawn. The backward
// pass is the same kernel on the incoming gradient. The mask depends on nothing
// but (seed, offset, row, col): not on the type, strides, launch shape or batch.
//
// Sixteen bits an element halve the integer work of the draw: ten rounds are 20
// wide multiplications, 2.5 an element here.
#include "b200_elem.cuh"
#include "b200_philox.cuh"
#include "b200_train.h"

namespace b200 {

struct DropoutArgs {
  const void* x;
  const void* residual;  // or null
  void* y;
  int64_t ldx, ldr, ldy;
  int K;
  unsigned units, units_per_row;  // of eight columns; units = rows * units_per_row < 2^31
  unsigned div_mul, div_shift;    // unit / units_per_row = (unit * div_mul) >> div_shift
  unsigned row0;                  // index of the first row (slices of one call)
  uint64_t seed, offset;
  const int64_t* offset_ptr;  // added to `offset` when given (read by the kernel)
  unsigned cut;
  float scale;
};

// The unit's random words. Element 2 w is the low half of word w, 2 w + 1 the high.
__device__ __forceinline__ void draw(uint32_t (&c)[4], const DropoutArgs& a, unsigned row, unsigned unit, uint64_t offset) {
  c[0] = unit;
  c[1] = row;
  c[2] = (uint32_t)offset;
  c[3] = (uint32_t)(offset >> 32);
  philox_4x32_10(c, a.seed);
}

// Aligned rows: a thread owns a unit at a time, 16-byte loads and stores. At 16-bit
// types a unit takes 120 instructions with its conversions: 8192 x 4096 bf16 27 us, which
// is 76 % of the measured memory rate with the SMs issuing 57 % of the time, so that neither
// is used up; a thread's load, draw and store follow one another. fp32: 48 us (5.5 TB/s), bound
// by memory. Two units a thread were slower (35 us for bf16: half the warps). `cut` is compared
// in the upper half of a word, so that the high halves need no shift.
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_vec_kernel(const DropoutArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const uint64_t offset = a.offset + (a.offset_ptr ? (uint64_t)*a.offset_ptr : 0ull);
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* res = reinterpret_cast<const T*>(a.residual);
  T* y = reinterpret_cast<T*>(a.y);
  const uint32_t cut = a.cut << 16;
  for (unsigned u = blockIdx.x * 256u + threadIdx.x; u < a.units; u += gridDim.x * 256u) {
    const unsigned row = (unsigned)(((uint64_t)u * a.div_mul) >> a.div_shift);
    const unsigned unit = u - row * a.units_per_row;
    const int64_t r = row, c = (int64_t)unit * 8;
    Group<T, 8> v, q;
    v.load(x + r * a.ldx + c);
    if (RES) q.load(res + r * a.ldr + c);
    uint32_t w[4];
    draw(w, a, a.row0 + row, unit, offset);
    float f[8], g[8];
    v.unpack(f);
    if (RES) q.unpack(g);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = (w[j] << 16) >= cut ? f[2 * j] * a.scale : 0.f;
      f[2 * j + 1] = w[j] >= cut ? f[2 * j + 1] * a.scale : 0.f;
    }
    if (RES) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += g[j];
    }
    v.pack(f);
    v.store(y + r * a.ldy + c);
  }
}

// Rows of any width, stride and alignment: a warp owns 256 columns. Each lane
// draws one unit's bits; the elements then go by column = lane + 32 j, so that
// every access of the warp is contiguous, with the bits fetched from their lane.
// 2047 x 5001 fp16 with a residual 17.5 us (3.5 TB/s), without 16 us: bound by
// instructions, an access being two bytes a lane (issuing 70 % of the time).
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_any_kernel(const DropoutArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const uint64_t offset = a.offset + (a.offset_ptr ? (uint64_t)*a.offset_ptr : 0ull);
  const int lane = threadIdx.x & 31;
  const uint32_t cut = a.cut << 16;
  // here a "unit" of the division is a warp's chunk of 256 columns
  for (unsigned u = blockIdx.x * 8u + (threadIdx.x >> 5); u < a.units; u += gridDim.x * 8u) {
    const unsigned row = (unsigned)(((uint64_t)u * a.div_mul) >> a.div_shift);
    const unsigned chunk = u - row * a.units_per_row;
    const int64_t r = row;
    const int c0 = (int)(chunk * 256u) + lane;
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.ldx + c0;
    const T* res = reinterpret_cast<const T*>(a.residual) + r * a.ldr + c0;
    T* y = reinterpret_cast<T*>(a.y) + r * a.ldy + c0;
    T v[8], q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + 32 * j < a.K) {
        v[j] = x[32 * j];
        if (RES) q[j] = res[32 * j];
      }
    uint32_t w[4];
    draw(w, a, a.row0 + row, chunk * 32u + lane, offset);
    unsigned bits = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) bits |= ((w[j] << 16) >= cut ? 1u << (2 * j) : 0u) | (w[j] >= cut ? 2u << (2 * j) : 0u);
    const unsigned mine = 1u << (lane & 7);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned b = __shfl_sync(0xffffffffu, bits, 4 * j + (lane >> 3));
      if (c0 + 32 * j < a.K) {
        float f = b & mine ? to_f32(v[j]) * a.scale : 0.f;
        if (RES) f += to_f32(q[j]);
        y[32 * j] = from_f32<T>(f);
      }
    }
  }
}

// n / d for n < 2^31 as (n * mul) >> shift, exact: mul = floor(2^(31+l) / d) + 1
// with 2^l >= d, so that 0 < mul * d - 2^(31+l) <= 2^l (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994).
static void magic_div(unsigned d, unsigned* mul, unsigned* shift) {
  unsigned l = 0;
  while ((1ull << l) < d) ++l;
  *shift = 31 + l;
  *mul = (unsigned)(((1ull << (31 + l)) / d) + 1);
}

template <typename T>
static int launch_dropout(DropoutArgs a, int64_t rows, bool vec, int num_sms, cudaStream_t st) {
  const int64_t upr = vec ? a.K / 8 : ((int64_t)a.K + 255) / 256;
  a.units_per_row = (unsigned)upr;
  magic_div(a.units_per_row, &a.div_mul, &a.div_shift);
  const int64_t slice = ((1ll << 31) - 1) / upr;  // rows a launch may number with 31 bits of units
  const char *x = (const char*)a.x, *r = (const char*)a.residual;
  char* y = (char*)a.y;
  for (int64_t r0 = 0; r0 < rows; r0 += slice) {
    const int64_t n = rows - r0 < slice ? rows - r0 : slice;
    a.x = x + r0 * a.ldx * (int64_t)sizeof(T);
    a.residual = r ? r + r0 * a.ldr * (int64_t)sizeof(T) : nullptr;
    a.y = y + r0 * a.ldy * (int64_t)sizeof(T);
    a.row0 = (unsigned)r0;
    a.units = (unsigned)(n * upr);
    const unsigned per = vec ? 256 : 8;
    unsigned grid = (a.units + per - 1) / per;
    const unsigned most = (unsigned)num_sms * 8;  // no more CTAs than can be resident
    grid = grid < most ? grid : most;
    void (*kernel)(const DropoutArgs) = vec ? (a.residual ? dropout_vec_kernel<T, true> : dropout_vec_kernel<T, false>)
                                            : (a.residual ? dropout_any_kernel<T, true> : dropout_any_kernel<T, false>);
    const cudaError_t e = launch_k(kernel, dim3(grid), dim3(256), 0, st, 1, a);
    if (e != cudaSuccess) return (int)e;
  }
  return (int)cudaGetLastError();
}

}  // namespace b200

using namespace b200;

extern "C" {

// y[rows, K] = dropout(x) (+ residual); strides in elements, type: ElemType of all
// three. 0 <= cut < 65536 (a call that drops everything needs no kernel).
// Returns 0, a CUDA error code, or -1 for arguments out of range.
int b200_dropout(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y, int64_t ldy, int64_t rows,
                 int K, int type, uint64_t seed, uint64_t offset, const int64_t* offset_ptr, int cut, float scale,
                 int num_sms, cudaStream_t st) {
  if (rows < 0 || K < 0 || K > 0x7FFFFE00 || rows > 0xFFFFFFFFll || cut < 0 || cut > 65535 || type < 0 || type > 2) return -1;
  if (rows == 0 || K == 0) return 0;
  DropoutArgs a = {};
  a.x = x;
  a.residual = residual;
  a.y = y;
  a.ldx = ldx;
  a.ldr = ldr;
  a.ldy = ldy;
  a.K = K;
  a.seed = seed;
  a.offset = offset;
  a.offset_ptr = offset_ptr;
  a.cut = (unsigned)cut;
  a.scale = scale;
  const int size = type == kElemF32 ? 4 : 2;
  auto aligned = [&](const void* p, int64_t ld) { return p == nullptr || (((uintptr_t)p | (uintptr_t)(ld * size)) & 15) == 0; };
  const bool vec = K % 8 == 0 && aligned(x, ldx) && aligned(residual, ldr) && aligned(y, ldy);
  if (type == kElemBf16) return launch_dropout<__nv_bfloat16>(a, rows, vec, num_sms, st);
  if (type == kElemF16) return launch_dropout<__half>(a, rows, vec, num_sms, st);
  return launch_dropout<float>(a, rows, vec, num_sms, st);
}

}  // extern "C"

B200_STATUS_ACCESSORS(dropout)
