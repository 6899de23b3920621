// Matrices into e4m3 with a scale for each block of 128 (gfx950):
//   * k_norm      h = x + r;  y = h / sqrt(mean(h^2) + eps) * w;  y in 1 x 128 blocks
//   * k_rows      x in 1 x 128 blocks
//   * k_tiles     x in 128 x 128 blocks
// All three are bound by HBM: each element is read once and written once (k_norm keeps its row
// in registers between the sum of squares and the conversion), and the conversion is the
// hardware's v_cvt_pk_fp8_f32 (to nearest, ties to even).
//
// A block's scale s comes from the largest finite magnitude a in it, q = e4m3(v * (1/s)):
//   float32  s = a / 448, at least 2^-126 (so that 1/s is finite)
//   e8m0     s = 2^p, the least p with a <= 448 * 2^p
// and s = 1 for a block of zeros. NaN and infinities become NaN and leave the scale alone.
#include "fp8_blocks.h"

namespace yoda_fp8 {
namespace {

constexpr int kWidth = 8;                        // neighbouring columns of one lane: 16 B of 16-bit input
constexpr int kLanes = kBlockK / kWidth;         // 16 lanes hold one block's row: one DPP row
constexpr int kXcds = 8;

// Largest value over the 16 lanes of a DPP row: neighbours, pairs, then the mirrored halves.
__device__ __forceinline__ float row_max(float v) {
  auto step = [](float x, int y) { return fmaxf(x, __int_as_float(y)); };
  v = step(v, __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, true));    // quad_perm [1,0,3,2]
  v = step(v, __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, true));    // quad_perm [2,3,0,1]
  v = step(v, __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, true));   // row_half_mirror
  v = step(v, __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true));   // row_mirror
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
  v = row_max(v);
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off);
  return v;
}

// |v| where it is finite, else 0
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.f;
}

// A block's scale and its inverse from its largest finite magnitude.
template <bool POW2>
__device__ __forceinline__ float scale_of(float amax) {
  if (!(amax > 0.f)) return 1.f;
  if constexpr (POW2) {
    // amax = m * 2^e with 1 <= m < 2, and 448 = 1.75 * 2^8: p = e - 8 where m <= 1.75, else e - 7.
    // A subnormal amax ends at the least exponent either way.
    const uint32_t b = __float_as_uint(amax);
    int p = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u);
    p = p < -126 ? -126 : p;
    return __uint_as_float((uint32_t)(p + 127) << 23);
  } else {
    return fmaxf(__fdiv_rn(amax, 448.f), 1.17549435e-38f);
  }
}

template <bool POW2>
__device__ __forceinline__ void put_scale(void* scales, int64_t at, float s) {
  if constexpr (POW2) ((uint8_t*)scales)[at] = (uint8_t)(__float_as_uint(s) >> 23);
  else ((float*)scales)[at] = s;
}

// Eight values times 1/s, as e4m3 bytes. |v * inv| <= 448 * (1 + 2^-22) for a block's finite
// values, which rounds to 448 at most; infinity times inv converts to NaN.
__device__ __forceinline__ uint2 to_e4m3(const float (&v)[kWidth], float inv) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// v, to nearest, where the exact value is v + rest: the neighbour with an odd last bit instead if rest is not 0.
// A later rounding to fewer bits is then that of the exact value.
__device__ __forceinline__ float to_odd(float v, float rest) {
  const int b = __float_as_int(v), step = (b ^ __float_as_int(rest)) >> 31 | 1;      // -1 toward 0, 1 away from it
  return __int_as_float(fabsf(rest) > 0.f && !(b & 1) ? b + step : b);        // (a NaN rest leaves v as it is)
}

// The first `keep` of eight bytes, zeros behind them.
__device__ __forceinline__ uint2 clear_past(uint2 v, int keep) {
  const uint64_t all = (uint64_t)v.y << 32 | v.x, kept = keep <= 0 ? 0 : all & (~0ull >> (64 - 8 * keep));
  return make_uint2((uint32_t)kept, (uint32_t)(kept >> 32));
}

// Eight neighbours of a row from column c on; zeros from column `cols` on. The rows of a caller's
// matrix start at any element, so the wide access assumes no more than an element's alignment.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int c, int cols, float (&v)[kWidth]) {
  using B = typename Bits<T>::type;
  if (c + kWidth <= cols) {
    const u32x4 a = Wide<sizeof(T)>::load(row + c);
    if constexpr (sizeof(T) == 4) {
      const u32x4 b = Wide<4>::load(row + c + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a[i]), v[4 + i] = __uint_as_float(b[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = load_f32<T>((uint16_t)(a[i] & 0xFFFF));
        v[2 * i + 1] = load_f32<T>((uint16_t)(a[i] >> 16));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kWidth; ++i) v[i] = c + i < cols ? load_f32<T>(((const B*)row)[c + i]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* row, int c, int cols, const float (&v)[kWidth]) {
  using B = typename Bits<T>::type;
  if (c + kWidth <= cols) {
    u32x4 a;
    if constexpr (sizeof(T) == 4) {
      u32x4 b;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = __float_as_uint(v[i]), b[i] = __float_as_uint(v[4 + i]);
      Wide<4>::store(row + c + 4, b);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
    Wide<sizeof(T)>::store(row + c, a);
  } else {
#pragma unroll
    for (int i = 0; i < kWidth; ++i)
      if (c + i < cols) ((B*)row)[c + i] = store_bits<T>(v[i]);
  }
}

// Workgroups go round the eight XCDs. Neighbouring rows write neighbouring scales, so each XCD
// gets a run of rows and its L2 joins their scales into whole lines. Returns -1 past the end.
__device__ __forceinline__ int64_t row_of(int64_t b, int64_t rows) {
  const int64_t run = (rows + kXcds - 1) / kXcds, at = b / kXcds, r = (b % kXcds) * run + at;
  return at < run && r < rows ? r : -1;
}

// A block of the norm in 64 bits, for what float32 cannot hold on the way: products h * w, a root or values out of
// (kLeast, kMost), a block of zeros, a row of NaN. (In float32 the factor root / s alone is infinite for a block
// whose products lie below 2^-119, and its zeros become NaN.) Neither h * w, which is exact, nor root / s leaves
// 64 bits' range. Returns the scale; all 16 lanes of the block come here together.
constexpr float kLeast = 1e-30f, kMost = 1e30f;

template <bool POW2>
__device__ __forceinline__ float wide_block(const float (&h)[kWidth], const float (&w)[kWidth], double root,
                                            float (&v)[kWidth]) {
  double amax = 0.;
#pragma unroll
  for (int i = 0; i < kWidth; ++i) {
    const double g = fabs((double)h[i] * w[i]);
    amax = g <= 1.7976931348623157e308 ? fmax(amax, g) : amax;
  }
#pragma unroll
  for (int off = 1; off < kLanes; off <<= 1) amax = fmax(amax, __shfl_xor(amax, off));
  amax *= root;                                  // NaN in the row, or 1/0: NaN, scale 1
  float s = 1.f;
  if (amax > 0.) {
    if constexpr (POW2) {
      const uint64_t b = (uint64_t)__double_as_longlong(amax);
      const int p = (int)(b >> 52) - 1023 - 8 + ((b & 0xFFFFFFFFFFFFFull) > 0xC000000000000ull);
      s = __uint_as_float((uint32_t)(min(max(p, -126), 127) + 127) << 23);
    } else {
      s = (float)fmin(fmax(amax / 448., 0x1p-126), 3.402823466e38);
    }
  }
  const double f = root / s;
#pragma unroll
  for (int i = 0; i < kWidth; ++i) {
    const double y = (double)h[i] * w[i] * f;
    v[i] = (float)y;
    v[i] = to_odd(v[i], (float)(y - v[i]));
  }
  return s;
}

struct NormArgs {
  const void *x, *residual, *weight;
  void *stream_out, *values, *scales;
  int64_t rows, x_pitch, r_pitch, s_pitch;   // pitches in elements
  int cols, padded;
  double eps;
};

// One workgroup a row. CHUNKS > 0: the row stays in registers (padded <= THREADS * CHUNKS * 8);
// CHUNKS == 0: the row is read twice (rows wider than that).
//
// Many rows: HBM. 16384 x 8192 in bf16 with a residual stream moves 940 MB in 186 us, 5.05 TB/s where a copy of 1 GB
// reaches 5.12; 512 or 1024 lanes a row, non-temporal loads and stores, and 32-bit sums were no faster.
// Few rows: the way of one row through load, sum, barrier, weight and store. From a graph, without a residual: 1 x 4096 3.1 us, 333 x 5001 5.3 on the same
// rows again and 7.1 on new ones (333 x 5120 4.9 and 6.6, 64 x 8192 4.4 and 5.0): what it takes beyond one row's is the
// way to memory, for two workgroups on a CU. Twice the lanes took 1 x 4096 with a residual from 4.5 to 3.6 us, 333 x 5001
// from 6.4 to 5.6 and 64 x 8192 from 7.3 to 5.1 up to 1024 rows
// (four a CU); with more they cost 3 % (4096 x 4096 30.7 : 31.3) to 5 % (2000 x 5001 14.6 : 15.3).
template <typename T, typename W, bool POW2, bool RES, int THREADS, int CHUNKS>
__global__ __launch_bounds__(THREADS) void k_norm(NormArgs a) {
  constexpr int kWaves = THREADS / 64;
  __shared__ double part[kWaves];
  const int64_t r = row_of(blockIdx.x, a.rows);
  if (r < 0) return;
  const T* x = (const T*)a.x + r * a.x_pitch;
  const T* res = RES ? (const T*)a.residual + r * a.r_pitch : nullptr;
  T* out = RES ? (T*)a.stream_out + r * (int64_t)a.cols : nullptr;
  const W* w = (const W*)a.weight;
  const int tid = threadIdx.x;
  const int chunks = CHUNKS ? CHUNKS : (a.padded + THREADS * kWidth - 1) / (THREADS * kWidth);

  // h of one chunk: the stream is rounded to its own type once, and the norm reads what it stores
  auto take = [&](int c, float (&h)[kWidth]) {
    load8<T>(x, c, a.cols, h);
    if constexpr (RES) {
      float o[kWidth];
      load8<T>(res, c, a.cols, o);
#pragma unroll
      for (int i = 0; i < kWidth; ++i) h[i] = load_f32<T>(store_bits<T>(h[i] + o[i]));
    }
  };

  // one chunk a lane: the weight is asked for with the row, not after the sum (1024 x 4096 10.3 -> 9.8 us)
  constexpr bool kEarly = CHUNKS == 1;
  float kept[CHUNKS ? CHUNKS : 1][kWidth], early[kWidth];
  double sum = 0.;
#pragma unroll
  for (int k = 0; k < chunks; ++k) {
    const int c = (k * THREADS + tid) * kWidth;
    float(&h)[kWidth] = kept[CHUNKS ? k : 0];
    if (c < a.padded) {
      if constexpr (kEarly) load8<W>(w, c, a.cols, early);
      take(c, h);
#pragma unroll
      for (int i = 0; i < kWidth; ++i) sum = fma((double)h[i], (double)h[i], sum);
    } else {
#pragma unroll
      for (int i = 0; i < kWidth; ++i) h[i] = 0.f;
    }
  }
  // squares, sums and the root in 64 bits: float32 would lose rows below 1e-19 and above 1e19, and it takes no longer
  double total = wave_sum(sum);
  if constexpr (kWaves > 1) {
    if ((tid & 63) == 0) part[tid >> 6] = total;
    __syncthreads();
    total = 0.;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) total += part[i];
  }
  const double root = 1. / sqrt(total / a.cols + a.eps);
  const float rstd = (float)root, rstd_low = (float)(root - rstd);

  uint8_t* q = (uint8_t*)a.values + r * (int64_t)a.padded;
#pragma unroll
  for (int k = 0; k < chunks; ++k) {
    const int c = (k * THREADS + tid) * kWidth;
    float again[kWidth];
    float(&h)[kWidth] = CHUNKS ? kept[CHUNKS ? k : 0] : again;
    if (c < a.padded) {          // the 16 lanes of a block agree: padded is a multiple of 128
      if constexpr (CHUNKS == 0) take(c, h);
      if constexpr (RES) store8<T>(out, c, a.cols, h);
      // Within a block the root cancels: with g = h * w, exact for 16-bit h and w,
      //   y / s = 448 g / max |g|,  or for a power of two  y / s = g * (rstd / s),
      // each with its first rounding's error added back and rounded to odd: the conversion that follows then
      // gives the 8-bit value next to the quotient itself, also where float32 would round onto a border.
      float g[kWidth], late[kWidth], v[kWidth], gmax = 0.f;
      const float(&w8)[kWidth] = kEarly ? early : late;
      if constexpr (!kEarly) load8<W>(w, c, a.cols, late);
#pragma unroll
      for (int i = 0; i < kWidth; ++i) {
        g[i] = h[i] * w8[i];
        gmax = fmaxf(gmax, fabsf(g[i]));               // (NaN counts for nothing)
      }
      gmax = row_max(gmax);
      if (!(gmax < kMost)) {                           // an infinite weight is left out, a product out of range is not
        gmax = 0.f;
#pragma unroll
        for (int i = 0; i < kWidth; ++i) gmax = fmaxf(gmax, fabsf(w8[i]) <= 3.402823466e38f ? fabsf(g[i]) : 0.f);
        gmax = row_max(gmax);
      }
      float amax = gmax * rstd;
      // a product that was rounded down onto 448 * 2^p lies above it
      if (POW2 && fmaf(gmax, rstd, -amax) + gmax * rstd_low > 0.f) amax = __uint_as_float(__float_as_uint(amax) + 1);
      float s;
      if (gmax > kLeast && gmax < kMost && rstd > kLeast && rstd < kMost && amax > kLeast && amax < kMost) {
        s = scale_of<POW2>(amax);
        if constexpr (!POW2) {
          const float inv = __fdiv_rn(1.f, gmax);
#pragma unroll
          for (int i = 0; i < kWidth; ++i) {
            const float top = g[i] * 448.f, first = top * inv;
            const float rest = fmaf(-first, gmax, top);
            v[i] = fabsf(rest) < 1e30f ? fmaf(rest, inv, first) : first;   // NaN and infinity as they are
            v[i] = to_odd(v[i], fmaf(-v[i], gmax, top));
          }
        } else {
          const float f = rstd * __fdiv_rn(1.f, s), low = rstd_low * __fdiv_rn(1.f, s);
#pragma unroll
          for (int i = 0; i < kWidth; ++i) {
            const float rest = g[i] * low;
            v[i] = fabsf(rest) < 1e30f ? fmaf(g[i], f, rest) : g[i] * f;
            v[i] = to_odd(v[i], fmaf(g[i], f, -v[i]) + rest);
          }
        }
      } else {
        s = wide_block<POW2>(h, w8, root, v);
      }
      uint2 out8 = to_e4m3(v, 1.f);
      if (c + kWidth > a.cols) out8 = clear_past(out8, a.cols - c);      // 0 * NaN in a padded column
      *(uint2*)(q + c) = out8;
      if (tid % kLanes == 0) put_scale<POW2>(a.scales, (int64_t)(c / kBlockK) * a.s_pitch + r, s);
    }
  }
}

struct QuantArgs {
  const void* x;
  void *values, *scales;
  int64_t rows, pitch, s_pitch;
  int cols, padded, lane_bits;         // 1 << lane_bits lanes a row and pass
};

constexpr int kThreads = 256;

// 1 x 128 blocks: a workgroup takes 256 >> lane_bits neighbouring rows. HBM: 8191 x 10240 in bf16 moves 253 MB in 49 us,
// 5.14 TB/s, a copy's rate; non-temporal loads and stores and 512 lanes were no faster.
template <typename T, bool POW2>
__global__ __launch_bounds__(kThreads) void k_rows(QuantArgs a) {
  const int per = kThreads >> a.lane_bits;
  const int64_t tiles = (a.rows + per - 1) / per, tile = row_of(blockIdx.x, tiles);
  if (tile < 0) return;
  const int64_t r = tile * per + (threadIdx.x >> a.lane_bits);
  if (r >= a.rows) return;             // whole 16-lane rows leave together: lane_bits >= 4
  const T* x = (const T*)a.x + r * a.pitch;
  uint8_t* q = (uint8_t*)a.values + r * (int64_t)a.padded;
  const int lane = threadIdx.x & ((1 << a.lane_bits) - 1);
  for (int c = lane * kWidth; c < a.padded; c += kWidth << a.lane_bits) {
    float v[kWidth], amax = 0.f;
    load8<T>(x, c, a.cols, v);
#pragma unroll
    for (int i = 0; i < kWidth; ++i) amax = fmaxf(amax, finite_abs(v[i]));
    const float s = scale_of<POW2>(row_max(amax));
    *(uint2*)(q + c) = to_e4m3(v, __fdiv_rn(1.f, s));
    if (threadIdx.x % kLanes == 0) put_scale<POW2>(a.scales, (int64_t)(c / kBlockK) * a.s_pitch + r, s);
  }
}

// 128 x 128 blocks: one workgroup a block, held in registers between the maximum and the conversion. HBM: 4096 x 4096
// in bf16 moves 50 MB in 10.5 us, 4.8 TB/s: four workgroups a CU in one round, which all load, then all store.
template <typename T, bool POW2>
__global__ __launch_bounds__(kThreads) void k_tiles(QuantArgs a) {
  constexpr int kRowsAtOnce = kThreads / kLanes, kPasses = kBlockK / kRowsAtOnce;
  __shared__ float part[kThreads / 64];
  const int kb = a.padded / kBlockK;
  const int64_t rb = blockIdx.x / kb;
  const int cb = (int)(blockIdx.x % kb), c = cb * kBlockK + (threadIdx.x % kLanes) * kWidth;
  const int64_t r0 = rb * kBlockK + threadIdx.x / kLanes;
  float v[kPasses][kWidth], amax = 0.f;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int64_t r = r0 + p * kRowsAtOnce;
    if (r < a.rows) {
      load8<T>((const T*)a.x + r * a.pitch, c, a.cols, v[p]);
    } else {
#pragma unroll
      for (int i = 0; i < kWidth; ++i) v[p][i] = 0.f;
    }
  }
#pragma unroll
  for (int p = 0; p < kPasses; ++p)
#pragma unroll
    for (int i = 0; i < kWidth; ++i) amax = fmaxf(amax, finite_abs(v[p][i]));
  amax = wave_max(amax);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 64; ++i) amax = fmaxf(amax, part[i]);
  const float s = scale_of<POW2>(amax), inv = __fdiv_rn(1.f, s);
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int64_t r = r0 + p * kRowsAtOnce;
    if (r < a.rows) *(uint2*)((uint8_t*)a.values + r * (int64_t)a.padded + c) = to_e4m3(v[p], inv);
  }
  if (threadIdx.x == 0) put_scale<POW2>(a.scales, rb * ((kb + 3) / 4 * 4) + cb, s);
}

int padded_cols(int cols) { return (cols + kBlockK - 1) / kBlockK * kBlockK; }

// A launch holds fewer than 2^32 threads, so a matrix goes in pieces of at most this many rows.
constexpr int64_t kRowsALaunch = 1 << 21;

template <typename T, typename W, bool POW2, bool RES>
int norm_piece(const NormArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)((a.rows + kXcds - 1) / kXcds * kXcds);
  const bool few = a.rows <= 1024;
#define YODA_NORM(threads, chunks) k_norm<T, W, POW2, RES, threads, chunks><<<grid, threads, 0, s>>>(a)
  if (a.padded <= 64 * 8) YODA_NORM(64, 1);
  else if (a.padded <= 128 * 8) YODA_NORM(128, 1);
  else if (a.padded <= 256 * 8) YODA_NORM(256, 1);
  else if (few && a.padded <= 512 * 8) YODA_NORM(512, 1);
  else if (a.padded <= 256 * 2 * 8) YODA_NORM(256, 2);
  else if (few && a.padded <= 512 * 2 * 8) YODA_NORM(512, 2);
  else if (a.padded <= 256 * 4 * 8) YODA_NORM(256, 4);
  else if (few && a.padded <= 1024 * 2 * 8) YODA_NORM(1024, 2);
  else if (a.padded <= 512 * 4 * 8) YODA_NORM(512, 4);
  else if (a.padded <= 1024 * 4 * 8) YODA_NORM(1024, 4);
  else YODA_NORM(1024, 0);
#undef YODA_NORM
  return (int)hipGetLastError();
}

template <typename T, typename W, bool POW2, bool RES>
int norm_sized(const NormArgs& all, hipStream_t s) {
  int rc = 0;
  for (int64_t at = 0; at < all.rows && !rc; at += kRowsALaunch) {
    NormArgs a = all;
    a.rows = all.rows - at < kRowsALaunch ? all.rows - at : kRowsALaunch;
    a.x = (const T*)all.x + at * all.x_pitch;
    if (RES) a.residual = (const T*)all.residual + at * all.r_pitch, a.stream_out = (T*)all.stream_out + at * all.cols;
    a.values = (uint8_t*)all.values + at * all.padded;
    a.scales = (uint8_t*)all.scales + at * (POW2 ? 1 : 4);
    rc = norm_piece<T, W, POW2, RES>(a, s);
  }
  return rc;
}

template <typename T, typename W>
int norm_typed(const NormArgs& a, bool pow2, hipStream_t s) {
  if (pow2) return a.residual ? norm_sized<T, W, true, true>(a, s) : norm_sized<T, W, true, false>(a, s);
  return a.residual ? norm_sized<T, W, false, true>(a, s) : norm_sized<T, W, false, false>(a, s);
}

template <typename T>
int quant_typed(const QuantArgs& all, bool tiles, bool pow2, hipStream_t s) {
  if (tiles) {
    const int64_t grid = (all.rows + kBlockK - 1) / kBlockK * (all.padded / kBlockK);
    if (grid >= 1 << 24) return -1;             // 2^32 threads; 256 GB of values
    if (pow2) k_tiles<T, true><<<(unsigned)grid, kThreads, 0, s>>>(all);
    else k_tiles<T, false><<<(unsigned)grid, kThreads, 0, s>>>(all);
  } else {
    for (int64_t at = 0; at < all.rows; at += kRowsALaunch) {
      QuantArgs a = all;
      a.rows = all.rows - at < kRowsALaunch ? all.rows - at : kRowsALaunch;
      a.x = (const T*)all.x + at * all.pitch;
      a.values = (uint8_t*)all.values + at * all.padded;
      a.scales = (uint8_t*)all.scales + at * (pow2 ? 1 : 4);
      const int64_t per = kThreads >> a.lane_bits, count = (a.rows + per - 1) / per;
      const unsigned grid = (unsigned)((count + kXcds - 1) / kXcds * kXcds);
      if (pow2) k_rows<T, true><<<grid, kThreads, 0, s>>>(a);
      else k_rows<T, false><<<grid, kThreads, 0, s>>>(a);
    }
  }
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace yoda_fp8

using namespace yoda_fp8;

extern "C" {

// x, residual: rows x cols of `type` with the pitches given (elements); weight: cols of `type` or
// float32 (weight_f32). stream_out (with a residual only): rows x cols, contiguous.
// Returns 0, a hipError, or -1 for arguments out of range.
int yoda_fp8_norm(int device, void* stream, int type, int weight_f32, int pow2, const void* x, int64_t x_pitch,
                  const void* residual, int64_t r_pitch, const void* weight, void* stream_out, void* values,
                  void* scales, int64_t rows, int cols, double eps) {
  if (!valid_type(type) || rows < 0 || rows > 0x7FFFFF00 || cols < 1 || cols > (1 << 30)) return -1;
  if ((residual == nullptr) != (stream_out == nullptr)) return -1;
  if (rows == 0) return 0;
  if (!x || !weight || !values || !scales) return -1;
  DeviceScope on(device);
  if (on.err != hipSuccess) return (int)on.err;
  const NormArgs a = {x, residual, weight, stream_out, values, scales, rows, x_pitch, r_pitch, (rows + 7) / 8 * 8, cols,
                      padded_cols(cols), eps};
  const hipStream_t s = (hipStream_t)stream;
  if (type == kFp32) return norm_typed<float, float>(a, pow2, s);
  if (type == kFp16) return weight_f32 ? norm_typed<__half, float>(a, pow2, s) : norm_typed<__half, __half>(a, pow2, s);
  return weight_f32 ? norm_typed<__hip_bfloat16, float>(a, pow2, s)
                    : norm_typed<__hip_bfloat16, __hip_bfloat16>(a, pow2, s);
}

// x: rows x cols of `type`, pitch in elements; tiles: 128 x 128 blocks, else 1 x 128.
int yoda_fp8_quantize(int device, void* stream, int type, int tiles, int pow2, const void* x, int64_t pitch,
                      void* values, void* scales, int64_t rows, int cols) {
  if (!valid_type(type) || rows < 0 || rows > 0x7FFFFF00 || cols < 1 || cols > (1 << 30)) return -1;
  if (rows == 0) return 0;
  if (!x || !values || !scales) return -1;
  DeviceScope on(device);
  if (on.err != hipSuccess) return (int)on.err;
  QuantArgs a = {x, values, scales, rows, pitch, (rows + 7) / 8 * 8, cols, padded_cols(cols), 4};
  while (a.lane_bits < 8 && (kWidth << a.lane_bits) < a.padded) ++a.lane_bits;
  const hipStream_t s = (hipStream_t)stream;
  if (type == kFp32) return quant_typed<float>(a, tiles, pow2, s);
  if (type == kFp16) return quant_typed<__half>(a, tiles, pow2, s);
  return quant_typed<__hip_bfloat16>(a, tiles, pow2, s);
}

}  // extern "C"
