// Matrix-core probe: the 8-bit linear layer of fp8_blocks.hip / fp8_matmul.hip on a card, checked value
// by value against plain vector code and timed. What the HBM probes do not reach: matrix instructions, 8-bit
// conversions, LDS and the loads into it. A card that computes wrongly there passes every memory check.
//
// The checkers share no arithmetic with the operators: one thread sums a value from its definition, in float64
// for the norm and the weight, and for the product with the bound that the operator's sums have (each
// eight neighbouring products lose less than 7 * 2^-13 of their largest; then float32, then bf16).
//
// They are plain on purpose and read from L2 what the operators keep in LDS. 4096 x 4096 x 4096 with ten repetitions
// takes 36 ms and 236 MB of the card: the product's check 33 ms (4 TFLOP/s of vector code), the norm's 0.5, the weight's
// 0.07, the comparison of two products 0.012; the operators themselves 0.03, 0.01 and 0.05.
#include "fp8_blocks.h"

#include <algorithm>

extern "C" {
int yoda_fp8_norm(int device, void* stream, int type, int weight_f32, int pow2, const void* x, int64_t x_pitch,
                  const void* residual, int64_t r_pitch, const void* weight, void* stream_out, void* values,
                  void* scales, int64_t rows, int cols, double eps);
int yoda_fp8_quantize(int device, void* stream, int type, int tiles, int pow2, const void* x, int64_t pitch,
                      void* values, void* scales, int64_t rows, int cols);
int64_t yoda_fp8_matmul_workspace(int64_t m, int64_t n, int kb, int pow2);
int yoda_fp8_matmul(int device, void* stream, int out_type, int pow2, const void* a, const void* sa, const void* b,
                    const void* sb, const void* bias, void* out, int64_t m, int64_t n, int kb, int64_t pitch,
                    int64_t sa_pitch, void* workspace, int64_t workspace_bytes);
}

namespace yoda_fp8 {
namespace {

constexpr double kEps = 1e-6;
enum Stage { kNorm, kWeight, kProduct, kUnstable, kStages };         // of the counts of wrong values

// about normal (a sum of four uniform values), from the element's place and the seed; bf16
__global__ __launch_bounds__(256) void k_values(uint16_t* out, int64_t n, uint32_t seed, float scale, float shift) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    uint64_t z = (uint64_t)i * 0x9E3779B97F4A7C15ull + seed * 0xD1B54A32D192ED03ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    z ^= z >> 31;
    const float u = (float)((z & 0xFFFF) + (z >> 16 & 0xFFFF) + (z >> 32 & 0xFFFF) + (z >> 48)) * (1.f / 65536.f) - 2.f;
    out[i] = store_bits<__hip_bfloat16>(u * 1.73f * scale + shift);
  }
}

// v to bf16, to nearest, ties to even, by whole numbers (the operators convert by an instruction)
__device__ uint16_t round_bf16(float v) {
  const uint32_t b = __float_as_uint(v);
  return (uint16_t)((b + 0x7FFF + (b >> 16 & 1)) >> 16);
}

__device__ double bf16(uint16_t v) { return (double)__uint_as_float((uint32_t)v << 16); }
__device__ double bf16(const uint16_t* p, int64_t i) { return (double)__uint_as_float((uint32_t)p[i] << 16); }

__device__ double e4m3(uint8_t b) {
  const int e = b >> 3 & 15, f = b & 7;
  const double v = e ? ldexp(8. + f, e - 10) : ldexp((double)f, -9);
  return (b & 127) == 127 ? nan("") : b & 128 ? -v : v;
}

template <bool POW2>
__device__ double scale_in(const void* s, int64_t at) {
  if constexpr (POW2) return ldexp(1., (int)((const uint8_t*)s)[at] - 127);
  else return (double)((const float*)s)[at];
}

// whether scale s is that of a block whose largest magnitude is amax, within 2^-20
template <bool POW2>
__device__ bool right_scale(double s, double amax) {
  if (!(amax > 0)) return s == 1.;
  const double r = amax / 448, t = ldexp(1., -20);
  return POW2 ? s >= r * (1 - t) && s < 2 * r * (1 + t) : fabs(s - r) <= r * t;
}

__device__ bool right_value(double q, double s, double y) {
  const double step = fmax(fabs(y) * 0.0625, s * 0x1p-10);
  return fabs(q * s - y) <= step * (1 + 0x1p-16) + fabs(y) * 0x1p-20;       // false for NaN
}

__device__ void count(unsigned long long* errors, unsigned bad) {
  for (int off = 32; off > 0; off >>= 1) bad += __shfl_xor(bad, off, 64);
  if ((threadIdx.x & 63) == 0 && bad) atomicAdd(errors, (unsigned long long)bad);
}

// a workgroup of 128 a block of a row: h = x + r rounded, y = h / rms(h) * gain
template <bool POW2>
__global__ __launch_bounds__(128) void k_check_norm(const uint16_t* x, const uint16_t* r, const uint16_t* gain,
                                                   const uint16_t* h, const uint8_t* q, const void* sa, int64_t pitch,
                                                   int64_t rows, int cols, unsigned long long* errors) {
  __shared__ double part[128];
  const int64_t m = blockIdx.y;
  const int t = threadIdx.x;
  const int64_t c = (int64_t)blockIdx.x * 128 + t;
  double sum = 0;
  for (int k = t; k < cols; k += 128) {
    const float v = (float)bf16(x, m * cols + k) + (float)bf16(r, m * cols + k);
    const double b = bf16(round_bf16(v));
    sum += b * b;
  }
  part[t] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < 128; ++i) sum += part[i];
  __syncthreads();
  const float v = (float)bf16(x, m * cols + c) + (float)bf16(r, m * cols + c);
  const uint16_t hb = round_bf16(v);
  const double y = bf16(hb) / sqrt(sum / cols + kEps) * bf16(gain, c);
  part[t] = fabs(y);
  __syncthreads();
  double amax = 0;
  for (int i = 0; i < 128; ++i) amax = fmax(amax, part[i]);
  const double s = scale_in<POW2>(sa, (int64_t)blockIdx.x * pitch + m);
  count(errors, !(right_scale<POW2>(s, amax) && right_value(e4m3(q[m * cols + c]), s, y) && h[m * cols + c] == hb));
}

// a workgroup of 256 a 128 x 128 block of the weight
template <bool POW2>
__global__ __launch_bounds__(256) void k_check_weight(const uint16_t* w, const uint8_t* q, const void* sb, int sb_pitch,
                                                     int64_t rows, int cols, unsigned long long* errors) {
  __shared__ double part[256];
  const int64_t n0 = (int64_t)blockIdx.y * 128, c = (int64_t)blockIdx.x * 128 + (threadIdx.x & 127);
  double amax = 0;
  for (int i = threadIdx.x >> 7; i < 128; i += 2) amax = fmax(amax, fabs(bf16(w, (n0 + i) * cols + c)));
  part[threadIdx.x] = amax;
  __syncthreads();
  for (int i = 0; i < 256; ++i) amax = fmax(amax, part[i]);
  const double s = scale_in<POW2>(sb, blockIdx.y * (int64_t)sb_pitch + blockIdx.x);
  unsigned bad = !right_scale<POW2>(s, amax);
  for (int i = threadIdx.x >> 7; i < 128; i += 2)
    bad += !right_value(e4m3(q[(n0 + i) * cols + c]), s, bf16(w, (n0 + i) * cols + c));
  count(errors, bad);
}

// one thread an output: float32 sums of eight products are exact enough beside the bound (their error is 2^-21 of it)
template <bool POW2>
__global__ __launch_bounds__(256) void k_check_product(const uint8_t* a, const void* sa, int64_t sa_pitch,
                                                      const uint8_t* b, const void* sb, int sb_pitch, const uint16_t* out,
                                                      int64_t cols, int inner, unsigned long long* errors) {
  const int64_t m = blockIdx.y, n = (int64_t)blockIdx.x * 256 + threadIdx.x;
  double want = 0, largest = 0, mass = 0;
  for (int kb = 0; kb < inner / 128; ++kb) {
    const double s = scale_in<POW2>(sa, kb * sa_pitch + m) * scale_in<POW2>(sb, n / 128 * sb_pitch + kb);
    float sum = 0, top = 0, abs = 0;
    for (int k = kb * 128; k < kb * 128 + 128; k += 8) {
      const uint2 u = *(const uint2*)(a + m * inner + k), v = *(const uint2*)(b + n * inner + k);
      float one = 0;
#define YODA_PAIR(w, i) __builtin_amdgcn_cvt_f32_fp8(w, i)
#define YODA_ADD(x, y, i)                                   \
  {                                                         \
    const float p = YODA_PAIR(x, i) * YODA_PAIR(y, i);      \
    sum += p, abs += fabsf(p), one = fmaxf(one, fabsf(p));  \
  }
      YODA_ADD(u.x, v.x, 0) YODA_ADD(u.x, v.x, 1) YODA_ADD(u.x, v.x, 2) YODA_ADD(u.x, v.x, 3)
      YODA_ADD(u.y, v.y, 0) YODA_ADD(u.y, v.y, 1) YODA_ADD(u.y, v.y, 2) YODA_ADD(u.y, v.y, 3)
#undef YODA_ADD
#undef YODA_PAIR
      top += one;
    }
    want += s * sum, largest += s * top, mass += s * abs;
  }
  const double room = largest * 7 * 0x1p-13 * (1 + 0x1p-10) + mass * (2 * (inner + 2) * 0x1p-24 + 0x1p-17);
  const double got = bf16(out, m * cols + n);
  count(errors, !(fabs(got - want) <= room + (fabs(want) + room) * 0x1p-8));
}

__global__ __launch_bounds__(256) void k_differ(const uint32_t* a, const uint32_t* b, int64_t words, unsigned long long* errors) {
  unsigned bad = 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) bad += a[i] != b[i];
  count(errors, bad);
}

// device memory and events that end with the call
struct Held {
  void* all[16];
  int count = 0;
  hipEvent_t events[2] = {nullptr, nullptr};
  hipError_t err = hipSuccess;
  template <typename T = uint8_t>
  T* take(int64_t bytes) {
    void* p = nullptr;
    if (err == hipSuccess) err = hipMalloc(&p, (size_t)(bytes + 15) / 16 * 16);
    if (p) all[count++] = p;
    return (T*)p;
  }
  ~Held() {
    for (int i = 0; i < count; ++i) (void)hipFree(all[i]);
    for (hipEvent_t e : events)
      if (e) (void)hipEventDestroy(e);
  }
};

template <bool POW2>
int check(int device, int64_t rows, int64_t cols, int inner, int iters, uint32_t seed, uint32_t verify_seed,
          double* tflops, unsigned long long* errors) {
  Held mem;
  const int kb = inner / 128, sb_pitch = (kb + 3) / 4 * 4;
  const int64_t sa_pitch = (rows + 7) / 8 * 8, xs = rows * inner, ws = cols * inner, os = rows * cols;
  uint16_t *x = mem.take<uint16_t>(2 * xs), *r = mem.take<uint16_t>(2 * xs), *gain = mem.take<uint16_t>(2 * inner),
           *h = mem.take<uint16_t>(2 * xs), *w = mem.take<uint16_t>(2 * ws), *out = mem.take<uint16_t>(2 * os),
           *again = mem.take<uint16_t>(2 * os);
  uint8_t *qa = mem.take(xs), *qb = mem.take(ws);
  void *sa = mem.take(4 * sa_pitch * kb), *sb = mem.take(4 * sb_pitch * (cols / 128));
  const int64_t room = yoda_fp8_matmul_workspace(rows, cols, kb, POW2);
  void* space = mem.take(room + 16);
  unsigned long long* bad = mem.take<unsigned long long>(8 * kStages);
  for (hipEvent_t& e : mem.events)
    if (mem.err == hipSuccess) mem.err = hipEventCreate(&e);
  if (mem.err != hipSuccess) return (int)mem.err;

  const float small = 1.f / sqrtf((float)inner);
  auto fill = [&](uint16_t* p, int64_t n, uint32_t s, float scale, float shift) { k_values<<<2048, 256>>>(p, n, s, scale, shift); };
  fill(x, xs, seed, 1.f, 0.f);
  fill(r, xs, seed + 1, 2.f, 0.f);
  fill(gain, inner, seed + 2, 0.1f, 1.f);
  fill(w, ws, seed + 3, small, 0.f);
  hipError_t e = hipMemset(bad, 0, 8 * kStages);
  if (e != hipSuccess) return (int)e;
  auto operands = [&] {
    const int rc = yoda_fp8_norm(device, nullptr, kBf16, 0, POW2, x, inner, r, inner, gain, h, qa, sa, rows, inner, kEps);
    return rc ? rc : yoda_fp8_quantize(device, nullptr, kBf16, 1, POW2, w, inner, qb, sb, cols, inner);
  };
  int rc = operands();
  auto product = [&](uint16_t* to) {
    return yoda_fp8_matmul(device, nullptr, kBf16, POW2, qa, sa, qb, sb, nullptr, to, rows, cols, kb, cols, sa_pitch,
                           room ? space : nullptr, room);
  };
  if (!rc) rc = product(out);
  if (rc) return rc;
  const bool other = verify_seed != seed;        // the checkers go by another layer: its inputs, and then its operands
  if (other) fill(x, xs, verify_seed, 1.f, 0.f), fill(w, ws, verify_seed + 3, small, 0.f);
  k_check_norm<POW2><<<dim3(kb, (unsigned)rows), 128>>>(x, r, gain, h, qa, sa, sa_pitch, rows, inner, bad + kNorm);
  k_check_weight<POW2><<<dim3(kb, (unsigned)(cols / 128)), 256>>>(w, qb, sb, sb_pitch, cols, inner, bad + kWeight);
  if (other && (rc = operands())) return rc;
  k_check_product<POW2><<<dim3((unsigned)(cols / 256), (unsigned)rows), 256>>>(qa, sa, sa_pitch, qb, sb, sb_pitch, out, cols,
                                                                             inner, bad + kProduct);
  float best = 0.f;
  for (int i = 0; i < iters && !rc; ++i) {       // the same product again: the same bits, and how long it takes
    if ((e = hipEventRecord(mem.events[0], nullptr)) != hipSuccess) return (int)e;
    rc = product(again);
    if ((e = hipEventRecord(mem.events[1], nullptr)) != hipSuccess) return (int)e;
    k_differ<<<1024, 256>>>((const uint32_t*)out, (const uint32_t*)again, os / 2, bad + kUnstable);
    if ((e = hipEventSynchronize(mem.events[1])) != hipSuccess) return (int)e;
    float ms = 0.f;
    if ((e = hipEventElapsedTime(&ms, mem.events[0], mem.events[1])) != hipSuccess) return (int)e;
    if (i == 0 || ms < best) best = ms;
  }
  if (rc) return rc;
  if ((e = hipMemcpy(errors, bad, 8 * kStages, hipMemcpyDeviceToHost)) != hipSuccess) return (int)e;
  *tflops = best > 0.f ? 2. * rows * cols * inner / best / 1e9 : 0.;
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace yoda_fp8

using namespace yoda_fp8;

extern "C" {

// Device memory that the check of these sizes takes, in bytes.
int64_t yoda_fp8_matrix_check_bytes(int64_t rows, int64_t cols, int inner) {
  return 7 * rows * inner + 3 * cols * inner + 4 * rows * cols + (rows + 8) * inner / 32 + cols * inner / 4096 +
         std::max(yoda_fp8_matmul_workspace(rows, cols, inner / 128, 0), yoda_fp8_matmul_workspace(rows, cols, inner / 128, 1)) +
         (1 << 20);
}

// Norm, weight and product of the sizes given (rows from 1 to 65535, cols a multiple of 256, inner of 128), every
// value checked, the product repeated iters times. errors[4]: wrong values of the norm, the weight and the product, and
// pairs of the product's values that changed; *tflops: the fastest product's rate. With another verify_seed every checker
// goes by the inputs or operands of that seed's layer and has to find them off. Returns 0, a hipError, or -1 for sizes out of range.
int yoda_fp8_matrix_check(int device, int64_t rows, int64_t cols, int inner, int iters, int pow2, unsigned seed,
                          unsigned verify_seed, double* tflops, unsigned long long* errors) {
  if (rows < 1 || rows > 65535 || cols < 256 || cols % 256 || cols > (1 << 22) || inner < 128 || inner % 128 ||
      inner > (1 << 16) || iters < 1)
    return -1;
  DeviceScope on(device);
  if (on.err != hipSuccess) return (int)on.err;
  return pow2 ? check<true>(device, rows, cols, inner, iters, seed, verify_seed, tflops, errors)
              : check<false>(device, rows, cols, inner, iters, seed, verify_seed, tflops, errors);
}

}  // extern "C"
