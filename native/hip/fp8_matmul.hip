// out[m][n] = sum over blocks kb of sa[m][kb] * sb[n / 128][kb] * sum over k in kb of a[m][k] * b[n][k], plus bias[n]
// a: M x K in e4m3, 1 x 128 blocks; b: N x K in e4m3, 128 x 128 blocks; out: bf16 or fp16.
//
// v_mfma_*_f8f6f4 adds eight neighbouring products in fixed point, each cut off below 2^-13 of the
// largest one's power of two, and then sums in float32 (measured: beside 2^16, 2^3 counts and 6 is
// lost within the eight, 2^-7 counts outside them). That is about 1.3e-5 of a result of normal
// inputs, against 1.7e-3 for a bf16 output's rounding; float32 outputs are not offered for it.
#include "fp8_blocks.h"

namespace yoda_fp8 {
namespace {

struct MatArgs {
  const uint8_t *a, *b;                // [M][Kp], [N][Kp]
  const void *sa, *sb;                 // [Kp/128][M], [ceil(N/128)][Kp/128]
  const void* bias;                    // [N] of the output's type, or null
  void* out;
  int64_t m, n, pitch;                 // pitch of out in elements
  int kb;                              // Kp / 128
};

__device__ __forceinline__ i32x8 load32(const uint8_t* p) {
  const i32x4 x = *(const i32x4*)p, y = *(const i32x4*)(p + 16);
  return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <bool POW2>
__device__ __forceinline__ float scale_at(const void* s, int64_t at) {
  if constexpr (POW2) {
    const uint32_t b = ((const uint8_t*)s)[at];
    return b == 255 ? __uint_as_float(0x7FC00000u) : b ? __uint_as_float(b << 23) : 5.877471754e-39f;
  } else {
    return ((const float*)s)[at];
  }
}

// One wave a 16 x 16 tile. The weight is the matrix instruction's first operand, so that the four
// sums of a lane are four neighbours n of one row m.
template <typename O, bool POW2>
__global__ __launch_bounds__(256) void k_simple(MatArgs p) {
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int64_t n0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16, m = (int64_t)blockIdx.y * 16 + c;
  if (n0 >= p.n) return;
  const int64_t kp = (int64_t)p.kb * kBlockK, bn = n0 + c < p.n ? n0 + c : p.n - 1, am = m < p.m ? m : p.m - 1;
  const uint8_t *a = p.a + am * kp + g * 32, *b = p.b + bn * kp + g * 32;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int kb = 0; kb < p.kb; ++kb) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const f32x4 t = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(load32(b + kb * kBlockK), load32(a + kb * kBlockK),
                                                                    zero, 0, 0, 0, 0, 0, 0);
    const float s = scale_at<POW2>(p.sa, (int64_t)kb * p.m + am) * scale_at<POW2>(p.sb, n0 / kBlockK * p.kb + kb);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(t[i], s, acc[i]);
  }
  if (m >= p.m) return;
  using B = typename Bits<O>::type;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = n0 + g * 4 + i;
    if (n >= p.n) continue;
    const float v = acc[i] + (p.bias ? load_f32<O>(((const B*)p.bias)[n]) : 0.f);
    ((B*)p.out)[m * p.pitch + n] = store_bits<O>(v);
  }
}

template <typename O>
int run(const MatArgs& p, bool pow2, hipStream_t s) {
  const int64_t gx = (p.n + 63) / 64, gy = (p.m + 15) / 16;
  if (gx > 0x7FFFFFFF || gy > 65535) return -1;
  const dim3 grid((unsigned)gx, (unsigned)gy);
  if (pow2) k_simple<O, true><<<grid, 256, 0, s>>>(p);
  else k_simple<O, false><<<grid, 256, 0, s>>>(p);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace yoda_fp8

using namespace yoda_fp8;

extern "C" {

// kb: blocks along K. pitch: elements between rows of out. Returns 0, a hipError, or -1 for
// arguments out of range.
int yoda_fp8_matmul(int device, void* stream, int out_type, int pow2, const void* a, const void* sa, const void* b,
                    const void* sb, const void* bias, void* out, int64_t m, int64_t n, int kb, int64_t pitch) {
  if ((out_type != kBf16 && out_type != kFp16) || m < 0 || n < 0 || kb < 1 || kb > (1 << 23) || pitch < n) return -1;
  if (m == 0 || n == 0) return 0;
  if (!a || !sa || !b || !sb || !out) return -1;
  DeviceScope on(device);
  if (on.err != hipSuccess) return (int)on.err;
  const MatArgs p = {(const uint8_t*)a, (const uint8_t*)b, sa, sb, bias, out, m, n, pitch, kb};
  const hipStream_t s = (hipStream_t)stream;
  if (out_type == kFp16) return run<__half>(p, pow2, s);
  return run<__hip_bfloat16>(p, pow2, s);
}

}  // extern "C"
