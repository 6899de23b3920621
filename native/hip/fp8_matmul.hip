// out[m][n] = sum over blocks kb of sa[m][kb] * sb[n / 128][kb] * sum over k in kb of a[m][k] * b[n][k], plus bias[n]
// a: M x K in e4m3, 1 x 128 blocks; b: N x K in e4m3, 128 x 128 blocks; out: bf16 or fp16.
//
// v_mfma_*_f8f6f4 adds eight neighbouring products in fixed point, each cut off below 2^-13 of the
// largest one's power of two, and then sums in float32 (measured: beside 2^16, 2^3 counts and 6 is
// lost within the eight, 2^-7 counts outside them). That is about 1.3e-5 of a result of normal
// inputs, against 1.7e-3 for a bf16 output's rounding; float32 outputs are not offered for it.
#include "fp8_blocks.h"

#include <algorithm>

namespace yoda_fp8 {
namespace {

struct MatArgs {
  const uint8_t *a, *b;                // [M][Kp], [N][Kp]
  const void *sa, *sb;                 // [Kp/128][sa_pitch], [ceil(N/128)][Kp/128 up to a multiple of 4]
  const void* bias;                    // [N] of the output's type, or null
  void* out;
  int64_t m, n, pitch, sa_pitch;       // pitch of out in elements; sa_pitch: m up to a multiple of 8
  int kb, sb_pitch;                    // Kp / 128, and up to a multiple of 4
};

// A launch holds fewer than 2^32 threads, 512 of them a workgroup at most.
constexpr int64_t kMostGroups = 1 << 22;

template <int I>
struct Index {
  static constexpr int value = I;
};
// f(0), f(1), ... f(N - 1) with their numbers known to the compiler
template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F& f) {
  if constexpr (I < N) {
    f(Index<I>{});
    each<N, I + 1>(f);
  }
}

// ---------------------------------------------------------------- tiles through LDS
//
// One workgroup a tile of BM x BN, 128 of K a step: each wave holds 16*MT rows m times 16*NT columns
// n of sums. Lane (c, g) = (lane % 16, lane / 16) has the rows m = c*MT + i of its wave (i < MT), so that one
// load brings its scales, and of column piece j the four columns that make, over two pieces and the
// four g, 32 neighbours: a store writes 64 bytes of a row, 16 from each g.
//
// Both tiles lie in LDS as rows of 128 bytes, 16 rows a piece in the order of the c that reads them.
// The eight 16-byte parts of a row are exchanged by part ^= (row / 2) % 8, so that sixteen lanes that are
// served at once meet sixteen different parts of 256 bytes (64 banks). The loads go from memory into LDS directly: lane
// l of a load fills part l % 8 of row l / 8, and takes the part of memory that belongs there.
__host__ __device__ __forceinline__ constexpr int column_of(int piece, int c) {
  return (piece >> 1) * 32 + (c >> 2) * 8 + (piece & 1) * 4 + (c & 3);
}

// Lane l's BYTES at base + voff + soff go to LDS at lds + BYTES * l. m0 holds lds: the compiler keeps no values of its own
// in it ("reserved", hence its warning), and the clobber tells it that what it sets there for an instruction of its own
// does not outlast the load.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int BYTES>
__device__ __forceinline__ void load_lds(u32x4 rsrc, uint32_t voff, uint32_t soff, uint32_t lds) {
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(voff), "s"(rsrc), "s"(soff)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

__device__ __forceinline__ u32x4 buffer_of(const void* base) {
  const uint64_t at = (uint64_t)base;
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((uint32_t)at);
  r[1] = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
  r[2] = 0xFFFFFFFFu;
  r[3] = 0x00020000u;
  return r;
}

// The buffer where there is something to load, and an empty one elsewhere: its loads are counted and waited for
// like the others, and fetch nothing. So no load of a loop is behind a branch.
__device__ __forceinline__ u32x4 if_any(u32x4 rsrc, bool any) {
  rsrc[2] = __builtin_amdgcn_readfirstlane(any ? 0xFFFFFFFFu : 0u);
  return rsrc;
}

__device__ __forceinline__ i32x8 join(const i32x4 (&v)[2]) {
  return __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
}

// I: which byte of xscales holds this piece's scale
template <int I>
__device__ __forceinline__ f32x4 mfma_scaled(i32x8 w, i32x8 x, f32x4 acc, uint32_t wscale, uint32_t xscales) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc, 0, 0, 0, (int)wscale, I, (int)xscales);
}

// The tile of a workgroup: each XCD gets a run of them, in columns of kGroup rows, so that what runs at one
// time on an XCD shares rows and columns in its L2. False past the end.
__device__ __forceinline__ bool tile_of(int block, int tiles_m, int tiles_n, int& tm, int& tn) {
  constexpr int kXcds = 8, kGroup = 4;
  const int total = tiles_m * tiles_n, run = (total + kXcds - 1) / kXcds;
  const int at = block / kXcds, t = (block % kXcds) * run + at;
  if (at >= run || t >= total) return false;
  const int per = kGroup * tiles_n, first = t / per * kGroup, rows = min(kGroup, tiles_m - first);
  tm = first + t % per % rows;
  tn = t % per / rows;
  return true;
}

// A lane's MT rows from m on; n: the wave's first column. Four pieces at a time, so that the two stores to a line of
// 128 bytes follow each other and reach memory as one (two pieces at a time wrote 49 MB instead of 34 for 4096 x 4096 x
// 4096 and took 62.1 us instead of 61.2; 8192 x 8192 x 8192 399 : 393).
template <int MT, int NT, typename O>
__device__ __forceinline__ void store_tile(const MatArgs& p, const f32x4 (&acc)[MT][NT], int64_t m, int64_t n, int g) {
  using B = typename Bits<O>::type;
  n += g * 8;                           // of pieces 2j and 2j + 1: columns 32 j .. 32 j + 7 from here
  if (m >= p.m) return;
  const int rows = (int)min((int64_t)MT, p.m - m);
#pragma unroll
  for (int four = 0; four < NT; four += 4) {
    const int64_t at = n + 16 * four;
    if (at >= p.n) break;
    float bias[16] = {};
    if (p.bias) {
#pragma unroll
      for (int r = 0; r < 16; ++r) bias[r] = load_f32<O>(((const B*)p.bias)[min(at + (r & 7) + 4 * (r & 8), p.n - 1)]);
    }
    B* out = (B*)p.out + m * p.pitch + at;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (i >= rows) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 u = acc[i][four + 2 * h], v = acc[i][four + 2 * h + 1];
        const float* add = bias + 8 * h;
        const int64_t left = p.n - at - 32 * h;
        if (left >= 8) {
          Wide<sizeof(B)>::store(out + 32 * h, u32x4{pack2<O>(u[0] + add[0], u[1] + add[1]), pack2<O>(u[2] + add[2], u[3] + add[3]),
                                                     pack2<O>(v[0] + add[4], v[1] + add[5]), pack2<O>(v[2] + add[6], v[3] + add[7])});
        } else {
#pragma unroll
          for (int r = 0; r < 7; ++r)
            if (r < left) out[32 * h + r] = store_bits<O>((r < 4 ? u[r & 3] : v[r & 3]) + add[r]);
        }
      }
      out += p.pitch;
    }
  }
}

// 256 x 256 for e8m0 scales with four waves of 128 x 128, one to a SIMD: the matrix instruction applies
// the scales, so the sums never leave the accumulation registers, and fewer bytes leave LDS than with
// eight waves of 128 x 64 (128 KB a step instead of 192 KB, at 128 B a cycle and 2048 cycles of products).
//
// A step is four quarters of 16 products: rows x0, x1 (four pieces of 16 each) times columns w0, w1.
// Each quarter reads from LDS what a later one needs and loads 16 KB of the step after the next
// into what every wave has read:
//            products   reads                       loads
//   Q0(k)    x0 w0      w1(k)                       x0(k+2)
//   Q1(k)    x0 w1      x1(k)                       w0(k+2)
//   Q2(k)    x1 w1      x0(k+1)                     w1(k+2)
//   Q3(k)    x1 w0      w0(k+1), piece by piece     x1(k+2), rows' scales(k+3)
// A load has six quarters (of 512 cycles) to arrive; every wave counts its own loads (4, 4, 4 and 5 a quarter)
// and waits for those that the quarter reads, and the barrier joins the waits of all four. What a
// quarter loads into was read a step before (x0: waited for by count at Q0; the others: their
// products have been issued).
//
// 8192 x 8192 x 8192: 381 to 404 us by card, 2.7 to 2.9 PFLOP/s (a library's product with one scale for each matrix: 355
// us), 4096 x 4096 x 4096: 53 to 55 us. The matrix units are busy 69 to 72 % of the time, at 1.93 GHz (the library's 84 %,
// at 1.76): the busier they are, the lower the card's clock. A step's reads and loads are 1536 cycles of LDS beside the 2048
// of its products. Two meetings a step, 2, 8 or 16 rows of tiles a column and
// non-temporal stores were no faster. The stores of a round of tiles are 5 us of the 100, at the memory's rate.
struct Quarters {
  static constexpr int BM = 256, BN = 256;
  static constexpr int kPart = 128 * kBlockK;                     // x0, x1, w0 or w1 of one step: 16 KB
  static constexpr int kStep = 4 * kPart, kScales = 2 * kStep;    // then 4 steps x 4 waves x 256 scales of rows
  static constexpr int kHeld = kScales + 4 * 4 * 256;             // and each wave's columns' scales of 256 steps
  static constexpr int kLds = kHeld + 4 * 256;
};

// wait for all but `left` of the wave's loads, then for the other waves
template <int LEFT>
__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <typename O>
__global__ __launch_bounds__(256, 1) void k_quarters(MatArgs p, int tiles_m, int tiles_n) {
  using Q = Quarters;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Q::kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4, wm = wave >> 1, wn = wave & 1;
  int tm, tn;
  if (!tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn)) return;
  const int64_t m0 = (int64_t)tm * Q::BM, n0 = (int64_t)tn * Q::BN, kp = (int64_t)p.kb * kBlockK;
  const int64_t m = m0 + wm * 128 + c * 8, n = n0 + wn * 128;
  const int last = p.kb - 1;

  // LDS rows of a part: 64 * wm + 16 * i + c holds the row that lane c reads as piece i, row
  // 128 * wm + 8 * c + 4 * part + i; the columns' likewise
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  const u32x4 rx = buffer_of(p.a + m0 * kp), rw = buffer_of(p.b + n0 * kp);
  uint32_t vx[8], vw[8];
#pragma unroll
  for (int part = 0; part < 2; ++part)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = (wave + 4 * i) * 8 + lane / 8;              // of the part, in LDS
      const int64_t xm = (row >> 6) * 128 + (row & 15) * 8 + part * 4 + (row >> 4 & 3);
      const int64_t wc = (row >> 6) * 128 + column_of(part * 4 + (row >> 4 & 3), row & 15);
      const int key = row >> 1 & 7;
      vx[part * 4 + i] = (uint32_t)(min(xm, p.m - 1 - m0) * kp + ((lane & 7) ^ key) * 16);
      vw[part * 4 + i] = (uint32_t)(min(wc, p.n - 1 - n0) * kp + ((lane & 7) ^ key) * 16);
    }
  const uint32_t vs = (uint32_t)min((int64_t)lane * 4, p.sa_pitch - 4 - m0);
  auto load_x = [&](int part, int i, int k) {
    load_lds<16>(if_any(rx, k <= last), vx[part * 4 + i], k * kBlockK,
                 base + (k & 1) * Q::kStep + part * Q::kPart + (wave + 4 * i) * 1024);
  };
  auto load_w = [&](int part, int i, int k) {
    load_lds<16>(if_any(rw, k <= last), vw[part * 4 + i], k * kBlockK,
                 base + (k & 1) * Q::kStep + (2 + part) * Q::kPart + (wave + 4 * i) * 1024);
  };
  auto load_s = [&](int k) {
    const u32x4 rs = buffer_of((const uint8_t*)p.sa + m0 + k * p.sa_pitch);
    load_lds<4>(if_any(rs, k <= last), vs, 0, base + Q::kScales + ((k & 3) * 4 + wave) * 256);
  };

  const int piece = (g ^ (c >> 1)) * 16;
  const uint8_t* lx = lds + (wm * 64 + c) * kBlockK;
  const uint8_t* lw = lds + 2 * Q::kPart + (wn * 64 + c) * kBlockK;
  const uint8_t* ls = lds + Q::kScales + wave * 256 + wm * 128 + c * 8;
  i32x4 x[8][2], w[8][2];            // [piece][half of its 32 bytes]
  auto read_x = [&](int k, int i, int h) {
    x[i][h] = *(const i32x4*)(lx + (k & 1) * Q::kStep + (i >> 2) * Q::kPart + (i & 3) * 16 * kBlockK + (h ? piece ^ 64 : piece));
  };
  auto read_w = [&](int k, int j, int h) {
    w[j][h] = *(const i32x4*)(lw + (k & 1) * Q::kStep + (j >> 2) * Q::kPart + (j & 3) * 16 * kBlockK + (h ? piece ^ 64 : piece));
  };

  // the columns' scales of 256 steps: four in each lane, by way of LDS like all else, so that the compiler sees no
  // load that it would wait for behind the others
  const uint8_t* sb = (const uint8_t*)p.sb + min(n0 + wn * 128, p.n - 1) / kBlockK * p.sb_pitch;
  auto load_columns = [&](int k) {
    load_lds<4>(buffer_of(sb + k), (uint32_t)min(lane, (last - k) >> 2) * 4, 0, base + Q::kHeld + wave * 256);
  };
  const uint32_t* held = (const uint32_t*)(lds + Q::kHeld + wave * 256) + lane;

  f32x4 acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto four = [&](auto load) {
#pragma unroll
    for (int i = 0; i < 4; ++i) load(i);
  };
  load_columns(0);
  load_s(0);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    four([&](int i) { load_x(0, i, k); });
    four([&](int i) { load_w(0, i, k); });
    four([&](int i) { load_w(1, i, k); });
    load_s(k + 1);
    four([&](int i) { load_x(1, i, k); });
  }
  meet<26>();
  uint32_t sbs = *held;
  uint2 next = *(const uint2*)ls, now;
#pragma unroll
  for (int i = 0; i < 4; ++i) read_x(0, i, 0), read_x(0, i, 1);
#pragma unroll
  for (int j = 0; j < 4; ++j) read_w(0, j, 0), read_w(0, j, 1);
  // Nothing is pending where the loop begins, so that in it the compiler waits for what it needs alone
  // (0xC07F: lgkmcnt 0, the other counters at their most).
  __builtin_amdgcn_s_waitcnt(0xC07F);

#pragma unroll 1
  for (int k = 0; k < p.kb; ++k) {
    if ((k & 255) == 0 && k) {
      load_columns(k);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      sbs = *held;
    }
    // product number `at` of a quarter, one piece of columns after the other
    auto quarter = [&](auto Rows, auto Cols, auto between) {
      constexpr int r = decltype(Rows)::value, q = decltype(Cols)::value;
      const uint32_t ws = __builtin_amdgcn_readlane(sbs, k >> 2 & 63) >> (8 * (k & 3));
      auto one = [&](auto At) {
        constexpr int at = decltype(At)::value, i = r * 4 + at % 4, j = q * 4 + at / 4;
        acc[i][j] = mfma_scaled<i & 3>(join(w[j]), join(x[i]), acc[i][j], ws, r ? now.y : now.x);
        between(at);
        __builtin_amdgcn_sched_barrier(0);
      };
      each<16>(one);
    };
    asm volatile("s_waitcnt lgkmcnt(8)" ::: "memory");            // x0(k) and the scales are in registers
    meet<22>();
    now = next;
    quarter(Index<0>{}, Index<0>{}, [&](int at) {
      if (at % 2 == 0) read_w(k, 4 + at / 4, at / 2 % 2);
      if (at % 4 == 1) load_x(0, at / 4, k + 2);
    });
    meet<21>();
    quarter(Index<0>{}, Index<1>{}, [&](int at) {
      if (at % 2 == 0) read_x(k, 4 + at / 4, at / 2 % 2);
      if (at % 4 == 1) load_w(0, at / 4, k + 2);
    });
    meet<21>();
    quarter(Index<1>{}, Index<1>{}, [&](int at) {
      if (at % 2 == 0) read_x(k + 1, at / 4, at / 2 % 2);
      if (at % 4 == 1) load_w(1, at / 4, k + 2);
    });
    meet<21>();
    next = *(const uint2*)(ls + (k + 1 & 3) * 1024);
    quarter(Index<1>{}, Index<0>{}, [&](int at) {
      if (at == 0) load_s(k + 3);
      if (at % 4 == 1) load_x(1, at / 4, k + 2);
      if (at % 4 == 3) read_w(k + 1, at / 4, 0);
      if (at % 4 == 0 && at) read_w(k + 1, at / 4 - 1, 1);
      if (at == 15) read_w(k + 1, 3, 1);
    });
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // nothing may reach LDS after the workgroup's end
  store_tile<8, 8, O>(p, acc, m, n, g);
}

// 256 x 256 for float scales with eight waves of 128 x 64, two to a SIMD. A block's sum leaves the matrix instruction
// and enters the float32 sum by a multiply-add with its scale, 4 of them to a product of 32 cycles: the
// vector units take half as long as the matrix units, next to them. The multiply-adds stay two products behind.
//
// A step is eight pieces of rows times four of columns. The next step's operands are read from LDS as
// registers fall free, and each part of LDS is filled again, for the step after the next, once every wave has read it:
//   piece 0 | 1 .. 4 | 5 6 7     "|": all waves meet; x[i] is read after piece i - 4, w[j] in piece 7
//   after the first meeting   w(k+2) and rows' pieces 0-3 (k+2)    (read in step k-1)
//   after the second          rows' pieces 4-7 (k+2), rows' scales (k+3)
// so a load has a step and a half to arrive. Each wave counts its own loads: 6 and 3.
//
// 4096 x 4096 x 4096: 58 to 61 us, 2.3 PFLOP/s, the matrix units busy 62 to 64 % of the time; 8192 x 8192 x 8192: 446 to 450.
// Bound as k_quarters is, with 192 KB a step read from LDS instead of
// 128: e8m0 scales take 53 us. (Four waves of 128 x 128 would hold 256 sums a lane, which leaves
// no vector registers for the multiply-adds.)
struct Eight {
  static constexpr int BM = 256, BN = 256;
  static constexpr int kRows = 128 * kBlockK;                     // half of the rows' pieces: 16 KB
  static constexpr int kStep = 4 * kRows, kScales = 2 * kStep;    // then 4 steps x 256 scales of rows
  static constexpr int kHeld = kScales + 4 * 1024;                // and each wave's columns' scales of 256 steps
  static constexpr int kLds = kHeld + 8 * 1024;
};

template <typename O>
__global__ __launch_bounds__(512, 2) void k_eight(MatArgs p, int tiles_m, int tiles_n) {
  using Q = Eight;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[Q::kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4, wm = wave >> 2, wn = wave & 3;
  int tm, tn;
  if (!tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn)) return;
  const int64_t m0 = (int64_t)tm * Q::BM, n0 = (int64_t)tn * Q::BN, kp = (int64_t)p.kb * kBlockK;
  const int64_t m = m0 + wm * 128 + c * 8, n = n0 + wn * 64;
  const int last = p.kb - 1;

  // LDS rows: rows' half h: 64 * wm + 16 * i + c holds row 128 * wm + 8 * c + 4 * h + i; columns: 64 * wn + 16 * j + c
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  const u32x4 rx = buffer_of(p.a + m0 * kp), rw = buffer_of(p.b + n0 * kp);
  uint32_t vx[4], vw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (wave + 8 * (i & 1)) * 8 + lane / 8;
    const int64_t at = (row >> 6) * 128 + (row & 15) * 8 + (i >> 1) * 4 + (row >> 4 & 3);
    vx[i] = (uint32_t)(min(at, p.m - 1 - m0) * kp + ((lane & 7) ^ (row >> 1 & 7)) * 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (wave + 8 * i) * 8 + lane / 8;
    const int64_t at = (row >> 6) * 64 + column_of(row >> 4 & 3, row & 15);
    vw[i] = (uint32_t)(min(at, p.n - 1 - n0) * kp + ((lane & 7) ^ (row >> 1 & 7)) * 16);
  }
  auto load_x = [&](int half, int i, int k) {
    load_lds<16>(if_any(rx, k <= last), vx[half * 2 + i], k * kBlockK,
                 base + (k & 1) * Q::kStep + half * Q::kRows + (wave + 8 * i) * 1024);
  };
  auto load_w = [&](int i, int k) {
    load_lds<16>(if_any(rw, k <= last), vw[i], k * kBlockK, base + (k & 1) * Q::kStep + 2 * Q::kRows + (wave + 8 * i) * 1024);
  };
  const uint32_t vs = (uint32_t)min((int64_t)(wave & 3) * 64 + lane, p.sa_pitch - 1 - m0) * 4;
  auto load_s = [&](int k) {                                      // waves 4-7 write the same once more
    const u32x4 rs = buffer_of((const float*)p.sa + m0 + k * p.sa_pitch);
    load_lds<4>(if_any(rs, k <= last), vs, 0, base + Q::kScales + (k & 3) * 1024 + (wave & 3) * 256);
  };

  const int piece = (g ^ (c >> 1)) * 16;
  const uint8_t* lx = lds + (wm * 64 + c) * kBlockK;
  const uint8_t* lw = lds + 2 * Q::kRows + (wn * 64 + c) * kBlockK;
  const uint8_t* ls = lds + Q::kScales + wm * 512 + c * 32;
  i32x4 x[4][2], w[4][2];            // [piece % 4][half of its 32 bytes]
  auto read_x = [&](int k, int i, int h) {
    x[i & 3][h] = *(const i32x4*)(lx + (k & 1) * Q::kStep + (i >> 2) * Q::kRows + (i & 3) * 16 * kBlockK + (h ? piece ^ 64 : piece));
  };
  auto read_w = [&](int k, int j, int h) {
    w[j][h] = *(const i32x4*)(lw + (k & 1) * Q::kStep + j * 16 * kBlockK + (h ? piece ^ 64 : piece));
  };

  // the columns' scales of 256 steps in LDS, of 64 of them one in each lane
  const float* sb = (const float*)p.sb + min(n, p.n - 1) / kBlockK * p.sb_pitch;
  auto load_columns = [&](int k, int i) {
    load_lds<4>(buffer_of(sb + k), (uint32_t)min(64 * i + lane, last - k) * 4, 0, base + Q::kHeld + wave * 1024 + i * 256);
  };
  const float* held = (const float*)(lds + Q::kHeld + wave * 1024) + lane;

  f32x4 acc[8][4], t[4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int i = 0; i < 4; ++i) load_columns(0, i);
  load_s(0), load_s(1);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) load_w(i, k);
    load_x(0, 0, k), load_x(0, 1, k);
    load_x(1, 0, k), load_x(1, 1, k);
    load_s(k + 2);
  }
  meet<12>();
  float sbs = held[0];
  f32x4 next[2] = {*(const f32x4*)ls, *(const f32x4*)(ls + 16)};
#pragma unroll
  for (int i = 0; i < 4; ++i) read_x(0, i, 0), read_x(0, i, 1);
#pragma unroll
  for (int j = 0; j < 4; ++j) read_w(0, j, 0), read_w(0, j, 1);
  __builtin_amdgcn_s_waitcnt(0xC07F);           // as in k_quarters

#pragma unroll 1
  for (int k = 0; k < p.kb; ++k) {
    if ((k & 63) == 0 && k) {
      if ((k & 255) == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load_columns(k, i);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      sbs = held[k & 192];
    }
    const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sbs), k & 63));
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = next[i >> 2][i & 3] * ws;
    auto add = [&](auto At) {
      constexpr int at = decltype(At)::value, i = at / 4, j = at % 4;
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(t[j][r], s[i], acc[i][j][r]);
    };
    auto one = [&](auto At) {
      constexpr int at = decltype(At)::value, i = at / 4, j = at % 4;
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      t[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(w[j]), join(x[i & 3]), zero, 0, 0, 0, 0, 0, 0);
      if constexpr (at >= 2) add(Index<at - 2>{});
      if constexpr (at == 3 || at == 19) {          // what is refilled after a meeting has left LDS in every wave
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        meet<9>();
      }
      if constexpr (i < 4) {
        if constexpr (j == 3) read_x(k, i + 4, 0), read_x(k, i + 4, 1);
      } else {
        if constexpr (j == 3) read_x(k + 1, i - 4, 0), read_x(k + 1, i - 4, 1);
        if constexpr (i == 7) read_w(k + 1, j, 0), read_w(k + 1, j, 1);
      }
      if constexpr (at == 5 || at == 7 || at == 9 || at == 11) load_w((at - 5) / 2, k + 2);
      if constexpr (at == 13 || at == 15) load_x(0, (at - 13) / 2, k + 2);
      if constexpr (at == 21 || at == 23) load_x(1, (at - 21) / 2, k + 2);
      if constexpr (at == 25) {
        load_s(k + 4);
        next[0] = *(const f32x4*)(ls + (k + 1 & 3) * 1024);
        next[1] = *(const f32x4*)(ls + (k + 1 & 3) * 1024 + 16);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    each<32>(one);
    add(Index<30>{});
    add(Index<31>{});
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // nothing may reach LDS after the workgroup's end
  store_tile<8, 4, O>(p, acc, m, n, g);
}

template <typename O>
int run_256(const MatArgs& p, bool pow2, hipStream_t s) {
  const int64_t tm = (p.m + 255) / 256, tn = (p.n + 255) / 256, total = tm * tn;
  if (total >= kMostGroups) return -1;          // 512 GB of output
  const unsigned grid = (unsigned)((total + 7) / 8 * 8);
  if (pow2) k_quarters<O><<<grid, 256, 0, s>>>(p, (int)tm, (int)tn);
  else k_eight<O><<<grid, 512, 0, s>>>(p, (int)tm, (int)tn);
  return (int)hipGetLastError();
}

// Four neighbours of row m from column n (a multiple of 4) on, plus bias.
template <typename O>
__device__ __forceinline__ void store4(const MatArgs& p, f32x4 v, int64_t m, int64_t n) {
  using B = typename Bits<O>::type;
  typedef uint32_t u32x2_at2 __attribute__((ext_vector_type(2), aligned(2)));
  B* out = (B*)p.out + m * p.pitch + n;
  if (p.bias) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += load_f32<O>(((const B*)p.bias)[min(n + r, p.n - 1)]);
  }
  if (n + 4 <= p.n) {
    *(u32x2_at2*)out = u32x2_at2{pack2<O>(v[0], v[1]), pack2<O>(v[2], v[3])};
  } else {
#pragma unroll
    for (int r = 0; r < 3; ++r)
      if (n + r < p.n) out[r] = store_bits<O>(v[r]);
  }
}

// ---------------------------------------------------------------- smaller tiles, K in parts
//
// For products with too few tiles of 256 x 256 to fill the card: four waves of 16*RP x 16*CP, two by two, and a ring of
// STAGES steps in LDS. 128 x 128 is for many rows; 128, 64 or 32 rows x 32 columns for one row of tiles: every workgroup
// reads all rows again (out of L2, 33 TB/s) and a piece of the weight (out of HBM) that nobody else reads.
// K is in gridDim.y parts, whose float32 sums go to a workspace and are joined by k_join in the order of the parts. Where two
// workgroups' stages fit in LDS, they share a CU and one runs while the other waits.
//
// 128 x 128: 0.44 us a step where the products take 0.21: 64 KB of reads and 32 KB of loads go through LDS.
// 777 x 5000 x 1928 takes 17 us, 0.88 PFLOP/s (280 tiles, so some CUs have two); 4096 x 2048 x 4096 34, 2.05 PFLOP/s.
// 256 x 128 by eight waves of 64 x 64 was no faster (17.5 and 34), by four of 128 x 64 slower (22 and 39).
// 128 x 32: 128 x 8192 x 4096 takes 14 us with float scales, 12 with e8m0, 2.6 TB/s: 256 workgroups, each of which
// starts, runs 32 steps of 0.26 us as its 20 KB a step arrive, and stores.
template <int RP_, int CP_>
struct Mid {
  static constexpr int RP = RP_, CP = CP_, BM = 32 * RP, BN = 32 * CP;
  static constexpr int kRows = BM * kBlockK, kColumns = BN * kBlockK;         // a step's bytes
  static constexpr int kStage = kRows + kColumns + 4 * 256;                   // and each wave's rows' scales
  static constexpr int kLoads = RP + CP + 1;                                  // of a wave and step
  static constexpr int kProducts = RP * CP, kSlots = kProducts > kLoads ? kProducts : kLoads;
};

// column c of piece j of CP: as in column_of where pieces pair up
template <int CP>
__device__ __forceinline__ constexpr int mid_column(int j, int c) {
  return CP == 1 ? c : column_of(j, c);
}

// (LDS is given at the launch: with its size in the kernel the compiler would reckon with one workgroup on a CU,
// spread the sums over the accumulation registers and move them to and fro every step.)
template <int RP, int CP, int STAGES, typename O, bool POW2>
__global__ __launch_bounds__(256, 2) void k_mid(MatArgs p, int tiles_m, int tiles_n, float* parts) {
  using Q = Mid<RP, CP>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4, wm = wave >> 1, wn = wave & 1;
  int tm, tn;
  if (!tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn)) return;
  const int64_t m0 = (int64_t)tm * Q::BM, n0 = (int64_t)tn * Q::BN, kp = (int64_t)p.kb * kBlockK;
  const int64_t m = m0 + wm * 16 * RP + c * RP, n = n0 + wn * 16 * CP;
  const int first = __builtin_amdgcn_readfirstlane((uint32_t)p.kb * blockIdx.y / gridDim.y);
  const int end = __builtin_amdgcn_readfirstlane((uint32_t)p.kb * (blockIdx.y + 1) / gridDim.y);

  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  const u32x4 rx = buffer_of(p.a + m0 * kp), rw = buffer_of(p.b + n0 * kp);
  uint32_t vx[RP], vw[CP];
#pragma unroll
  for (int i = 0; i < RP; ++i) {
    const int row = (wave + 4 * i) * 8 + lane / 8, half = row / (16 * RP), piece = row / 16 % RP;
    const int64_t at = half * 16 * RP + (row & 15) * RP + piece;
    vx[i] = (uint32_t)(min(at, p.m - 1 - m0) * kp + ((lane & 7) ^ (row >> 1 & 7)) * 16);
  }
#pragma unroll
  for (int i = 0; i < CP; ++i) {
    const int row = (wave + 4 * i) * 8 + lane / 8, half = row / (16 * CP), piece = row / 16 % CP;
    const int64_t at = half * 16 * CP + mid_column<CP>(piece, row & 15);
    vw[i] = (uint32_t)(min(at, p.n - 1 - n0) * kp + ((lane & 7) ^ (row >> 1 & 7)) * 16);
  }
  constexpr int kScale = POW2 ? 1 : 4;
  // rows' scales: bytes from the tile's first row on, or 64 floats from the wave's first row (of 128) or the tile's
  const int from = RP == 4 && !POW2 ? wm * 64 : 0;
  const uint32_t vs = POW2 ? (uint32_t)min((int64_t)lane * 4, p.sa_pitch - 4 - m0)
                           : (uint32_t)min((int64_t)from + lane, p.sa_pitch - 1 - m0) * 4;
  // load number i of a step's
  auto load = [&](int i, int k, int stage) {
    const uint32_t to = base + stage * Q::kStage;
    if (i < RP) {
      load_lds<16>(if_any(rx, k < end), vx[i < RP ? i : 0], k * kBlockK, to + (wave + 4 * i) * 1024);
    } else if (i < RP + CP) {
      load_lds<16>(if_any(rw, k < end), vw[i - RP], k * kBlockK, to + Q::kRows + (wave + 4 * (i - RP)) * 1024);
    } else {
      const u32x4 rs = buffer_of((const uint8_t*)p.sa + (m0 + k * p.sa_pitch) * kScale);
      load_lds<4>(if_any(rs, k < end), vs, 0, to + Q::kRows + Q::kColumns + wave * 256);
    }
  };

  const int piece = (g ^ (c >> 1)) * 16;
  const uint8_t* lx = lds + (wm * 16 * RP + c) * kBlockK;
  const uint8_t* lw = lds + Q::kRows + (wn * 16 * CP + c) * kBlockK;
  const uint8_t* ls = lds + Q::kRows + Q::kColumns + wave * 256 + (wm * 16 * RP - from + c * RP) * kScale;

  // the columns' scale of a step, by scalar loads (address space 4): four bytes, or a float
  typedef const uint32_t __attribute__((address_space(4))) * Scalars;
  const Scalars sb = (Scalars)((const uint8_t*)p.sb + min(n, p.n - 1) / kBlockK * p.sb_pitch * kScale);
  auto column_scale = [&](int k) { return POW2 ? sb[k >> 2] >> (8 * (k & 3)) : sb[k]; };

  f32x4 acc[RP][CP];
#pragma unroll
  for (int i = 0; i < RP; ++i)
#pragma unroll
    for (int j = 0; j < CP; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int d = 0; d < STAGES; ++d)
#pragma unroll
    for (int i = 0; i < Q::kLoads; ++i) load(i, first + d, d);
  // operands of two steps: one in use, one being read
  struct Step {
    i32x4 x[RP][2], w[CP][2];
    float s[RP];
    uint32_t b, c;
  } step[2];
  // read number `at`: the rows' pieces, the columns', the rows' scales
  auto read = [&](Step& to, int stage, int at) {
    const int h = (at & 1 ? piece ^ 64 : piece);
    if (at < 2 * RP) {
      to.x[at / 2][at & 1] = *(const i32x4*)(lx + stage + at / 2 * 16 * kBlockK + h);
    } else if (at < 2 * (RP + CP)) {
      to.w[at / 2 - RP][at & 1] = *(const i32x4*)(lw + stage + (at / 2 - RP) * 16 * kBlockK + h);
    } else if constexpr (POW2) {
      if constexpr (RP == 4) to.b = *(const uint32_t*)(ls + stage);
      else if constexpr (RP == 2) to.b = *(const uint16_t*)(ls + stage);
      else to.b = ls[stage];
    } else {
#pragma unroll
      for (int i = 0; i < RP; ++i) to.s[i] = ((const float*)(ls + stage))[i];
    }
  };
  meet<(STAGES - 1) * Q::kLoads>();
#pragma unroll
  for (int at = 0; at <= 2 * (RP + CP); ++at) read(step[0], 0, at);
  step[0].c = column_scale(first);

  int stage = 0;                                // step k's
  auto one_step = [&](int k, const Step& now, Step& next) {
    // step k is in this wave's registers, and after the meeting in every wave's; step k + 1 is in LDS
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    meet<(STAGES - 2) * Q::kLoads>();
    const int ahead = stage + 1 < STAGES ? stage + 1 : 0, bytes = ahead * Q::kStage, free = stage;
    stage = ahead;
    next.c = column_scale(min(k + 1, end - 1));
    f32x4 t[4];
    float s[RP];
    if constexpr (!POW2) {
#pragma unroll
      for (int i = 0; i < RP; ++i) s[i] = now.s[i] * __uint_as_float(now.c);
    }
    auto add = [&](auto At) {
      constexpr int at = decltype(At)::value, j = at / RP, i = at % RP;
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(t[at & 3][r], s[i], acc[i][j][r]);
    };
    auto one = [&](auto At) {
      constexpr int at = decltype(At)::value;
      if constexpr (at < Q::kProducts) {
        constexpr int j = at / RP, i = at % RP;
        if constexpr (POW2) {
          acc[i][j] = mfma_scaled<i>(join(now.w[j]), join(now.x[i]), acc[i][j], now.c, now.b);
        } else {
          const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
          t[at & 3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(now.w[j]), join(now.x[i]), zero, 0, 0, 0, 0, 0, 0);
        }
      }
      if constexpr (!POW2 && at >= 2 && at - 2 < Q::kProducts) add(Index<at - 2>{});
      // the reads come early, so that they are done when the step ends
      if (at < RP + CP) read(next, bytes, 2 * at), read(next, bytes, 2 * at + 1);
      if (at == RP + CP) read(next, bytes, 2 * at);
      if (at < Q::kLoads) load(at, k + STAGES, free);
      __builtin_amdgcn_sched_barrier(0);
    };
    each<Q::kSlots>(one);
    if constexpr (!POW2) {
      if constexpr (Q::kSlots - 2 < Q::kProducts) add(Index<Q::kSlots - 2>{});
      if constexpr (Q::kSlots - 1 < Q::kProducts) add(Index<Q::kSlots - 1>{});
    }
  };
#pragma unroll 1
  for (int k = first; k + 1 < end; k += 2) {
    one_step(k, step[0], step[1]);
    one_step(k + 1, step[1], step[0]);
  }
  if ((end - first) & 1) one_step(end - 1, step[0], step[1]);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // nothing may reach LDS after the workgroup's end
  if (parts) {
    // this part's sums as they lie in the registers: each store a whole KB
    f32x4* out = (f32x4*)parts + (((int64_t)blockIdx.y * tiles_m * tiles_n + (int64_t)tm * tiles_n + tn) * 4 + wave) * (RP * CP * 64) + lane;
#pragma unroll
    for (int i = 0; i < RP; ++i)
#pragma unroll
      for (int j = 0; j < CP; ++j) out[(i * CP + j) * 64] = acc[i][j];
  } else if constexpr (CP == 1) {
#pragma unroll
    for (int i = 0; i < RP; ++i)
      if (m + i < p.m && n + g * 4 < p.n) store4<O>(p, acc[i][0], m + i, n + g * 4);
  } else {
    store_tile<RP, CP, O>(p, acc, m, n, g);
  }
}

// out = the sum of the parts in their order, plus bias: four neighbours a lane, a tile every RP * CP workgroups. The parts
// come out of the caches; what it costs is a launch, about 2.5 us with the parts' stores.
template <int RP, int CP, typename O>
__global__ __launch_bounds__(256) void k_join(MatArgs p, int tiles_m, int tiles_n, const f32x4* parts, int count) {
  const int tile = blockIdx.x / (RP * CP), at = blockIdx.x % (RP * CP) * 256 + threadIdx.x;
  const int wave = at / (RP * CP * 64), i = at / 64 / CP % RP, j = at / 64 % CP, c = at & 15, g = at >> 4 & 3;
  const int64_t m = (int64_t)(tile / tiles_n) * (32 * RP) + (wave >> 1) * 16 * RP + c * RP + i;
  const int64_t n = (int64_t)(tile % tiles_n) * (32 * CP) + (wave & 1) * 16 * CP +
                    (CP == 1 ? g * 4 : (j >> 1) * 32 + g * 8 + (j & 1) * 4);
  if (m >= p.m || n >= p.n) return;
  const f32x4* in = parts + (int64_t)tile * (RP * CP * 256) + at;
  const int64_t apart = (int64_t)tiles_m * tiles_n * (RP * CP * 256);
  f32x4 v = in[0];
  for (int k = 1; k < count; ++k) v += in[k * apart];
  store4<O>(p, v, m, n);
}

template <int RP, int CP, int STAGES, typename O>
int run_mid(const MatArgs& p, bool pow2, int count, float* parts, hipStream_t s) {
  using Q = Mid<RP, CP>;
  const int64_t tm = (p.m + Q::BM - 1) / Q::BM, tn = (p.n + Q::BN - 1) / Q::BN, total = tm * tn;
  const dim3 grid((unsigned)((total + 7) / 8 * 8), count);
  float* to = count > 1 ? parts : nullptr;
  if (pow2) k_mid<RP, CP, STAGES, O, true><<<grid, 256, STAGES * Q::kStage, s>>>(p, (int)tm, (int)tn, to);
  else k_mid<RP, CP, STAGES, O, false><<<grid, 256, STAGES * Q::kStage, s>>>(p, (int)tm, (int)tn, to);
  if (count > 1) k_join<RP, CP, O><<<(unsigned)(total * RP * CP), 256, 0, s>>>(p, (int)tm, (int)tn, (const f32x4*)parts, count);
  return (int)hipGetLastError();
}

// ---------------------------------------------------------------- few rows
//
// Up to 16 rows the weight's bytes are what counts: one workgroup takes all rows and 16 * NP columns, its waves
// take every WAVES-th block of K and read their operands from memory straight into registers, DEPTH
// blocks ahead, each weight byte once on the whole card; the rows are read again by each workgroup, out of L2.
// No wave waits for another until the end, when the waves' sums are added through LDS in the order of
// the waves. Lane (c, g) has row c; columns as in column_of where NP is 2.
// 16 x 8192 x 8192 takes 13.6 us, 5.0 TB/s of the 6.1 that reads reach; 1 x 4096 x 4096 5.2, of which 2.8 are the
// bytes at that rate and the rest a launch. Tiles through LDS take 14.9 for the former.
template <int NP, int WAVES, int DEPTH, typename O, bool POW2>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4) void k_narrow(MatArgs p) {
  __shared__ f32x4 part[WAVES * NP * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16 * NP, kp = (int64_t)p.kb * kBlockK;
  const uint8_t *px = p.a + min((int64_t)c, p.m - 1) * kp + g * 16, *pw[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) pw[j] = p.b + min(n0 + (NP == 2 ? column_of(j, c) : c), p.n - 1) * kp + g * 16;
  const int64_t sa_at = min((int64_t)c, p.sa_pitch - 1), sb_at = n0 / kBlockK * p.sb_pitch;

  struct Block {
    i32x4 x[2], w[NP][2];
    float xs, ws;
    uint32_t xb, wb;
  };
  auto load = [&](Block& b, int kb) {
    const int64_t at = (int64_t)kb * kBlockK;
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) b.w[j][h] = *(const i32x4*)(pw[j] + at + 64 * h);
#pragma unroll
    for (int h = 0; h < 2; ++h) b.x[h] = *(const i32x4*)(px + at + 64 * h);
    const int64_t s = kb * p.sa_pitch + sa_at;
    if constexpr (POW2) {
      b.xb = ((const uint8_t*)p.sa)[s];
      b.wb = ((const uint8_t*)p.sb)[sb_at + kb];
    } else {
      b.xs = ((const float*)p.sa)[s];
      b.ws = ((const float*)p.sb)[sb_at + kb];
    }
  };

  f32x4 acc[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto use = [&](const Block& b) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      if constexpr (POW2) {
        acc[j] = mfma_scaled<0>(join(b.w[j]), join(b.x), acc[j], b.wb, b.xb);
      } else {
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        const f32x4 t = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(b.w[j]), join(b.x), zero, 0, 0, 0, 0, 0, 0);
        const float s = b.xs * b.ws;
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[j][r] = fmaf(t[r], s, acc[j][r]);
      }
    }
  };

  // Rows a power of two apart lie on one memory channel, so workgroups that walk K in step would ask few
  // channels at a time: each begins at a block of its own and goes round.
  const int first = blockIdx.x % p.kb;
  auto block = [&](int q) {
    const int kb = min(q, p.kb - 1) + first;
    return kb < p.kb ? kb : kb - p.kb;
  };
  Block ring[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) {
    load(ring[d], block(wave + d * WAVES));     // past the end: the last one, not used
    __builtin_amdgcn_sched_barrier(0);
  }
  int q = wave;
#pragma unroll 1
  for (; q + (2 * DEPTH - 1) * WAVES < p.kb; q += DEPTH * WAVES) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      use(ring[d]);
      load(ring[d], block(q + (d + DEPTH) * WAVES));
      __builtin_amdgcn_sched_barrier(0);        // or all DEPTH loads end up behind all uses, and are waited for at once
    }
  }
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) {
    if (q + d * WAVES < p.kb) use(ring[d]);
    if (q + (d + DEPTH) * WAVES < p.kb) load(ring[d], block(q + (d + DEPTH) * WAVES));
  }
#pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d)
    if (q + (d + DEPTH) * WAVES < p.kb) use(ring[d]);

#pragma unroll
  for (int j = 0; j < NP; ++j) part[(wave * NP + j) * 64 + lane] = acc[j];
  __syncthreads();
  for (int e = threadIdx.x; e < NP * 64; e += 64 * WAVES) {
    f32x4 v = part[e];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += part[w * NP * 64 + e];
    const int l = e & 63, j = e / 64;
    const int64_t m = l & 15, n = n0 + (NP == 2 ? (l >> 4) * 8 + j * 4 : (l >> 4) * 4);
    if (m < p.m && n < p.n) store4<O>(p, v, m, n);
  }
}

template <int NP, int WAVES, int DEPTH, typename O>
int narrow(const MatArgs& p, bool pow2, hipStream_t s) {
  const unsigned grid = (unsigned)((p.n + 16 * NP - 1) / (16 * NP));
  if (pow2) k_narrow<NP, WAVES, DEPTH, O, true><<<grid, 64 * WAVES, 0, s>>>(p);
  else k_narrow<NP, WAVES, DEPTH, O, false><<<grid, 64 * WAVES, 0, s>>>(p);
  return (int)hipGetLastError();
}

// ---------------------------------------------------------------- which one
//
// By sizes alone, the least of the estimates below, in us, fitted to what the kernels take on an MI355X:
//   up to 16 rows   2 + (weight + rows for every 32 columns) / 8 MB, and 3 for every further round of 256 workgroups
//   small tiles     up to 256 workgroups 5 + `one` a step, else 2 + (`round` + `two` a step) a round of 512, and no
//                   less than 3 + weight / 5.3 MB; K in parts: 2.5 more, and twice the parts' bytes / 5 MB
//   256 x 256       (10.5 + 1.4 a step, float scales 1.57) a round of 256; a last round of a share f counts (1 + f) / 2
// (They order the kinds; a time itself may be off by a quarter: 777 x 5000 x 1928 comes out as 21 us and takes 17, few rows
// times few columns, whose workgroups are too few to draw the card's whole rate, as less than they take.)
// Measured, this one : the next best, e8m0 scales: 16 x 8192 x 8192 few rows 13.4 : 14.9 32 x 32;
// 32 x 8192 x 8192 32 x 32 14.7 : 16.1 64 x 32; 64 x 8192 x 8192 64 x 32 15.3 : 16.7 64 x 64; 128 x 8192 x 4096 128 x 32
// 12 : 15 128 x 128 in two parts; 2048 x 2048 x 4096 128 x 128 23 : 44 256 x 256; 4096 x 4096 x 4096 256 x 256
// 53 : 64 128 x 128.
struct Shape {
  int rows, columns;                    // pieces of 32
  double one, two, round;               // us a step alone on a CU, of two on a CU; and a round's own
  double one_f, two_f;                  // with float scales
};
constexpr Shape kShapes[] = {
    {4, 4, 0.44, 0.90, 4.5, 0.50, 0.95},
    {4, 1, 0.215, 0.40, 2.5, 0.26, 0.45},
    {2, 1, 0.16, 0.28, 2.5, 0.20, 0.33},
    {1, 1, 0.15, 0.25, 2.5, 0.155, 0.25},
};

struct Plan {
  enum { kNarrow, kSmall, k256 } kind;
  int shape, parts;
  int64_t groups, bytes;                // workgroups; bytes of workspace
  double us;
  int64_t split;                        // columns from 0 on that tiles of 256 x 256 take before
};

double round_of_256(int kb, bool pow2) { return 10.5 + kb * (pow2 ? 1.4 : 1.57); }

Plan one_kind(int64_t m, int64_t n, int kb, bool pow2) {
  const double weight = (double)n * kb * kBlockK;
  Plan best = {Plan::k256, 0, 1, 0, 0, 0, 0};
  const int64_t big = (m + 255) / 256 * ((n + 255) / 256);
  const double rest = big % 256 ? (1 + big % 256 / 256.0) / 2 : 0;
  double least = std::max<double>(big / 256 + rest, 1) * round_of_256(kb, pow2);
  if (m <= 16 && n < kMostGroups * 32) {
    const double t = 2 + weight * 1.5 / 8e6 + 3. * ((n + 8191) / 8192 - 1);
    if (t < least) least = t, best = {Plan::kNarrow, 0, 1, 0, 0, 0, 0};
  }
  for (int shape = 0; shape < 4; ++shape) {
    const Shape& h = kShapes[shape];
    const int64_t tiles = (m + 32 * h.rows - 1) / (32 * h.rows) * ((n + 32 * h.columns - 1) / (32 * h.columns));
    for (int parts = 1; parts <= 16 && parts * 2 <= std::max(kb, 2); parts *= 2) {
      const int64_t groups = tiles * parts, bytes = parts > 1 ? groups * h.rows * h.columns * 4096 : 0;
      if ((parts > 1 && groups > 512) || groups >= kMostGroups) break;
      const int steps = (kb + parts - 1) / parts;
      const double rounds = (double)((groups + 511) / 512);
      double t = groups <= 256 ? 5 + steps * (pow2 ? h.one : h.one_f) : 2 + rounds * (h.round + steps * (pow2 ? h.two : h.two_f));
      t = std::max(t, 3 + weight / 5.3e6);
      if (parts > 1) t += 2.5 + 2 * bytes / 5e6;
      if (t < least) least = t, best = {Plan::kSmall, shape, parts, groups, bytes, 0, 0};
    }
  }
  best.us = least;
  return best;
}

Plan plan(int64_t m, int64_t n, int kb, bool pow2) {
  Plan best = one_kind(m, n, kb, pow2);
  // Tiles of 256 x 256 for as many whole rounds as there are, and what else suits the columns that are left: 4608 x 4096 x
  // 4096 takes 73 us instead of 93, 4096 x 4100 x 900 29 instead of 38, 4096 x 10240 x 4096 148 instead of 153.
  const int64_t tm = (m + 255) / 256, tn = (n + 255) / 256, most = tm * tn / 256 * 256 / tm;
  if (most < 1 || most >= tn) return best;
  Plan rest = one_kind(m, n - 256 * most, kb, pow2);
  rest.us += 2 + (double)((tm * most + 255) / 256) * round_of_256(kb, pow2);
  rest.split = 256 * most;
  return rest.kind != Plan::k256 && rest.us < best.us ? rest : best;
}

template <typename O>
int run(MatArgs p, bool pow2, float* workspace, int64_t bytes, hipStream_t s) {
  const Plan to = plan(p.m, p.n, p.kb, pow2);
  if (to.bytes > bytes || (to.bytes && !workspace)) return -1;
  if (to.split) {
    MatArgs first = p;
    first.n = to.split;
    if (const int rc = run_256<O>(first, pow2, s)) return rc;
    p.n -= to.split;
    p.b += to.split * p.kb * kBlockK;
    p.sb = (const uint8_t*)p.sb + to.split / kBlockK * p.sb_pitch * (pow2 ? 1 : 4);
    p.out = (uint16_t*)p.out + to.split;
    if (p.bias) p.bias = (const uint16_t*)p.bias + to.split;
  }
  if (to.kind == Plan::k256) return run_256<O>(p, pow2, s);
  // two pieces of columns a workgroup halve what is read of the rows, where that leaves enough workgroups
  if (to.kind == Plan::kNarrow) return p.n >= 8192 ? narrow<2, 8, 4, O>(p, pow2, s) : narrow<1, 8, 4, O>(p, pow2, s);
  // stages: those of one workgroup fill LDS where there is one on a CU, else those of two
  const bool alone = to.groups <= 256;
  if (to.shape == 0) return alone ? run_mid<4, 4, 4, O>(p, pow2, to.parts, workspace, s) : run_mid<4, 4, 2, O>(p, pow2, to.parts, workspace, s);
  if (to.shape == 1) return alone ? run_mid<4, 1, 6, O>(p, pow2, to.parts, workspace, s) : run_mid<4, 1, 3, O>(p, pow2, to.parts, workspace, s);
  if (to.shape == 2) return run_mid<2, 1, 5, O>(p, pow2, to.parts, workspace, s);
  return run_mid<1, 1, 8, O>(p, pow2, to.parts, workspace, s);
}

}  // namespace
}  // namespace yoda_fp8

using namespace yoda_fp8;

extern "C" {

// Bytes of workspace that a product of these sizes needs (16-byte aligned, its own for the length of the call).
int64_t yoda_fp8_matmul_workspace(int64_t m, int64_t n, int kb, int pow2) {
  return m < 1 || n < 1 || kb < 1 ? 0 : plan(m, n, kb, pow2).bytes;
}

// kb: blocks along K. pitch: elements between rows of out. sa_pitch: scales between a's blocks along K,
// a multiple of 8. Rows of values and scales are 16-byte aligned. Returns 0, a hipError, or -1 for arguments
// out of range.
int yoda_fp8_matmul(int device, void* stream, int out_type, int pow2, const void* a, const void* sa, const void* b,
                    const void* sb, const void* bias, void* out, int64_t m, int64_t n, int kb, int64_t pitch,
                    int64_t sa_pitch, void* workspace, int64_t workspace_bytes) {
  if ((out_type != kBf16 && out_type != kFp16) || m < 0 || n < 0 || kb < 1 || kb > 65535 || pitch < n || sa_pitch < m ||
      sa_pitch % 8)
    return -1;
  if (m == 0 || n == 0) return 0;
  if (!a || !sa || !b || !sb || !out) return -1;
  DeviceScope on(device);
  if (on.err != hipSuccess) return (int)on.err;
  const MatArgs p = {(const uint8_t*)a, (const uint8_t*)b, sa, sb, bias, out, m, n, pitch, sa_pitch, kb, (kb + 3) / 4 * 4};
  const hipStream_t s = (hipStream_t)stream;
  float* ws = (float*)workspace;
  if (out_type == kFp16) return run<__half>(p, pow2, ws, workspace_bytes, s);
  return run<__hip_bfloat16>(p, pow2, ws, workspace_bytes, s);
}

}  // extern "C"
