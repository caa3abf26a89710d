// Rotary positions on int16 rows, forward and backward (nsrl_rotary_rows).
//
// A pair (x0, x1) at position p turns by the angle a = p * turn, kept as a
// 64-bit fraction of a turn, so the product wraps where the angle does and far
// positions keep every bit.  cos and sin come from the nearest of 1,024 points
// of the circle and the remaining angle d (|d| <= 2^-11 turn = 0.0031 rad):
// cos d = 1 - d^2 / 2 within 4e-12, sin d = d within 5e-9, both below 2^-27.
//
// Bound by memory (2 bytes in and 2 out per element) as long as integer
// instructions are few: both integer pipes issue every other cycle.  So
//  - the angles are worked out once per (row, pair) into shared memory and
//    read by every head;
//  - a Q30 factor is c = 2^15 ch + cl with |cl| <= 2^14, and
//      rhu(x0 c - x1 s, 30) = (P + (Q >> 15)) >> 15,
//      P = x0 ch - x1 sh,  Q = x0 cl - x1 sl + 2^29,
//    exact in 32 bits (floor of a floor; |P| < 2^31 as c^2 + s^2 = 2^60,
//    |Q| < 2^31): five multiply-adds and a shift, where the 64-bit sum of two
//    widening products takes seven instructions.  An amplitude above 1 keeps
//    the 64-bit form;
//  - a thread keeps its column (head and pairs) and steps down the rows.
// The loads of a thread's first rows are under way while it works out angles.
//
// 65,536 rows of 8 x 64 take 32 us, 4.2 TB/s: 64% of copy bandwidth, half of the
// instructions for the angles.  A table of all 1,024 points (one load in place of
// two, from 64 cache lines in place of 8) took 32.4, two or four angles of a thread
// at once 32.4, 8 rows a thread no less, 48 registers 36.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace nsrl {
namespace {

__device__ const int32_t d_quarter_lut[257] = {NSRL_QUARTER_LUT_VALUES};

constexpr int MAX_THREADS = 256;
constexpr int MAX_PAIRS = 1024;  // (row, pair) angles of a block: 16 KB of shared memory
constexpr int AHEAD = 2;         // rows a thread loads ahead
constexpr int ROWS = 4;          // rows a thread takes, where there are enough

struct RotArgs {
  const int16_t* x;
  int16_t* y;
  long long ldx, ldy, rows;
  const unsigned long long* turns;
  const int32_t* positions;
  unsigned seq_len;
  int heads, hd, half, backward, amplitude;
  int block_rows;         // rows of a block
  int turning, per_head;  // items of a head that turn, and all of them (out of place: dims that pass through too)
  int per_row, down;      // items of a row; rows the block takes at once
  int step, along;        // blockDim.x = step * half + along
  unsigned by_row, by_head, by_half;  // ceil(2^22 / d) of the three divisors
};

// n / d for n < 1024 by m = ceil(2^22 / d): exact while n d < 2^22, and 0 for larger d.
__device__ __forceinline__ int small_div(unsigned n, unsigned m) { return (int)((n * m) >> 22); }

__device__ __forceinline__ long long mad_wide(int x, int y, long long z) {
  long long r;
  asm("mad.wide.s32 %0, %1, %2, %3;" : "=l"(r) : "r"(x), "r"(y), "l"(z));
  return r;
}

// Q30 cosine and sine of a 2^-64 turn (the integer recipe of nsrl_b200.h).
__device__ __forceinline__ void cos_sin_q30(unsigned long long a, int amplitude, int& c, int& s) {
  const unsigned n = (unsigned)((a + (1ull << 53)) >> 54);  // nearest point, 0..1024 (wraps in the sum)
  const long long d = (long long)(a - ((unsigned long long)n << 54));
  const int i = n & 255;
  const int lo = d_quarter_lut[i], hi = d_quarter_lut[256 - i];
  const bool odd = n & 256, neg = n & 512;  // quadrants 1 and 3; 2 and 3
  int S0 = odd ? hi : lo, C0 = odd ? -lo : hi;
  if (neg) {
    S0 = -S0;
    C0 = -C0;
  }
  const int r = __mulhi((int)(d >> 22), 1686629713);
  const int h256 = ((__mulhi(r, r) + (1 << 14)) >> 15) << 8;  // below 2^21
  const long long half = 1ll << 37;
  c = C0 - (int)(mad_wide(C0, h256, mad_wide(S0, r, half)) >> 38);
  s = S0 - (int)(mad_wide(S0, h256, mad_wide(C0, -r, half)) >> 38);
  if (amplitude != (1 << 30)) {
    // |c| may pass 2^30 by one, so an amplitude near 2 may reach 2^31: held to 2^31 - 1
    c = (int)max(-2147483647ll, min(2147483647ll, ((long long)c * amplitude + (1ll << 29)) >> 30));
    s = (int)max(-2147483647ll, min(2147483647ll, ((long long)s * amplitude + (1ll << 29)) >> 30));
  }
}

// rhu(x0 * c - x1 * s, 30) (MINUS) or rhu(x0 * c + x1 * s, 30), not yet saturated.
template <bool WIDE, bool MINUS>
__device__ __forceinline__ int turn(int x0, int ch, int cl, int x1, int sh, int sl) {
  if (WIDE) return (int)(mad_wide(x0, ch, mad_wide(MINUS ? -x1 : x1, sh, 1ll << 29)) >> 30);
  const int p = MINUS ? x0 * ch - x1 * sh : x0 * ch + x1 * sh;
  const int q = MINUS ? (x0 * cl + (1 << 29)) - x1 * sl : (x0 * cl + (1 << 29)) + x1 * sl;
  int r;
  asm("mad.hi.s32 %0, %1, %2, %3;" : "=r"(r) : "r"(q), "r"(1 << 17), "r"(p));  // p + (q >> 15)
  return r >> 15;
}

// VEC: an item is 16 dims of a head (8 pairs, or 16 dims past rotary_dim),
// two 16-byte accesses.  Otherwise an item is one pair, or one dim past rotary_dim.
template <bool VEC, bool INTERLEAVED, bool WIDE>
__global__ void __launch_bounds__(MAX_THREADS) rotary_kernel(const RotArgs a) {
  extern __shared__ __align__(16) int32_t angles[];  // [4][rows][half]: ch, cl, sh, sl (WIDE: c, s in the first two)
  const int angle_count = a.block_rows * a.half;
  int32_t* const ch = angles;
  int32_t* const cl = angles + angle_count;  // WIDE: s
  int32_t* const sh = angles + 2 * angle_count;
  int32_t* const sl = angles + 3 * angle_count;
  const long long row0 = (long long)blockIdx.x * a.block_rows;
  const int rows = (int)min((long long)a.block_rows, a.rows - row0);
  const int turning = a.turning, per_head = a.per_head, per_row = a.per_row, down = a.down;
  const int my_row = small_div(threadIdx.x, a.by_row);  // beyond `down`: this thread has no column

  griddep_wait();
  griddep_launch();
  const int16_t* const x = a.x + row0 * a.ldx;
  int16_t* const y = a.y + row0 * a.ldy;
  // element offsets of a column's two accesses within a row, and its first pair (-1: passes through)
  auto place = [&](int column, int head, int& i0, int& i1) -> int {
    const int slot = column - head * per_head, base = head * a.hd;
    if (slot < turning) {
      const int pair = VEC ? 8 * slot : slot;
      i0 = base + (INTERLEAVED ? 2 * pair : pair);
      i1 = INTERLEAVED ? i0 + (VEC ? 8 : 1) : i0 + a.half;
      return pair;
    }
    i0 = base + 2 * a.half + (VEC ? 16 : 1) * (slot - turning);
    i1 = i0 + (VEC ? 8 : 0);
    return -1;
  };
  auto load = [&](const int16_t* row, int i0, int i1, uint4& u0, uint4& u1) {
    if (VEC) {
      u0 = *reinterpret_cast<const uint4*>(row + i0);
      u1 = *reinterpret_cast<const uint4*>(row + i1);
    } else {
      u0.x = (uint32_t)(uint16_t)row[i0];
      u1.x = (uint32_t)(uint16_t)row[i1];
    }
  };

  int column = my_row < down ? threadIdx.x - my_row * per_row : per_row;
  int i0 = 0, i1 = 0, pair = -1;
  uint4 v0[AHEAD], v1[AHEAD];
  if (column < per_row) {
    pair = place(column, small_div(column, a.by_head), i0, i1);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (my_row + k * down < rows) load(x + (my_row + k * down) * a.ldx, i0, i1, v0[k], v1[k]);
  }
  {
    int row = small_div(threadIdx.x, a.by_half), p = threadIdx.x - row * a.half;
    for (int i = threadIdx.x; i < rows * a.half; i += blockDim.x) {
      const long long r = row0 + row;
      const long long at = a.positions ? (long long)a.positions[r] : (long long)((unsigned)r % a.seq_len);
      int c, s;
      cos_sin_q30((unsigned long long)at * a.turns[p], a.amplitude, c, s);
      if (a.backward) s = -s;
      if (WIDE) {
        ch[i] = c;
        cl[i] = s;
      } else {
        const int h = (c + (1 << 14)) >> 15, g = (s + (1 << 14)) >> 15;
        ch[i] = h;
        cl[i] = c - (h << 15);
        sh[i] = g;
        sl[i] = s - (g << 15);
      }
      row += a.step;
      p += a.along;
      if (p >= a.half) {
        p -= a.half;
        ++row;
      }
    }
  }
  __syncthreads();

  for (bool first = true; column < per_row; column += blockDim.x, first = false) {
    if (!first) pair = place(column, column / per_head, i0, i1);
    const int16_t* xr = x + my_row * a.ldx;
    int16_t* yr = y + my_row * a.ldy;
    int angle = my_row * a.half + pair;
    for (int r = my_row; r < rows; r += AHEAD * down) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (r + k * down >= rows) break;
        if (!first || r != my_row) load(xr, i0, i1, v0[k], v1[k]);  // past the rows loaded ahead
        if (VEC) {
          uint4 o0 = v0[k], o1 = v1[k];
          if (pair >= 0) {
            int e[16], t0[8], t1[8];
            unpack8(v0[k], *reinterpret_cast<int(*)[8]>(e));
            unpack8(v1[k], *reinterpret_cast<int(*)[8]>(e + 8));
#pragma unroll
            for (int q = 0; q < 8; q += 4) {
              int f[4][4];
#pragma unroll
              for (int j = 0; j < (WIDE ? 2 : 4); ++j)
                *reinterpret_cast<int4*>(f[j]) = *reinterpret_cast<const int4*>(angles + j * angle_count + angle + q);
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                const int i = q + m;
                const int x0 = e[INTERLEAVED ? 2 * i : i], x1 = e[INTERLEAVED ? 2 * i + 1 : 8 + i];
                if (WIDE) {
                  t0[i] = turn<true, true>(x0, f[0][m], 0, x1, f[1][m], 0);
                  t1[i] = turn<true, false>(x0, f[1][m], 0, x1, f[0][m], 0);
                } else {
                  t0[i] = turn<false, true>(x0, f[0][m], f[1][m], x1, f[2][m], f[3][m]);
                  t1[i] = turn<false, false>(x0, f[2][m], f[3][m], x1, f[0][m], f[1][m]);
                }
              }
            }
            if (INTERLEAVED) {
              o0 = make_uint4(pack_sat16(t1[0], t0[0]), pack_sat16(t1[1], t0[1]), pack_sat16(t1[2], t0[2]),
                              pack_sat16(t1[3], t0[3]));
              o1 = make_uint4(pack_sat16(t1[4], t0[4]), pack_sat16(t1[5], t0[5]), pack_sat16(t1[6], t0[6]),
                              pack_sat16(t1[7], t0[7]));
            } else {
              o0 = make_uint4(pack_sat16(t0[1], t0[0]), pack_sat16(t0[3], t0[2]), pack_sat16(t0[5], t0[4]),
                              pack_sat16(t0[7], t0[6]));
              o1 = make_uint4(pack_sat16(t1[1], t1[0]), pack_sat16(t1[3], t1[2]), pack_sat16(t1[5], t1[4]),
                              pack_sat16(t1[7], t1[6]));
            }
          }
          *reinterpret_cast<uint4*>(yr + i0) = o0;
          *reinterpret_cast<uint4*>(yr + i1) = o1;
        } else {
          const int x0 = (int)(int16_t)v0[k].x, x1 = (int)(int16_t)v1[k].x;
          if (pair < 0) {
            yr[i0] = (int16_t)x0;
          } else if (WIDE) {
            yr[i0] = (int16_t)sat16(turn<true, true>(x0, ch[angle], 0, x1, cl[angle], 0));
            yr[i1] = (int16_t)sat16(turn<true, false>(x0, cl[angle], 0, x1, ch[angle], 0));
          } else {
            yr[i0] = (int16_t)sat16(turn<false, true>(x0, ch[angle], cl[angle], x1, sh[angle], sl[angle]));
            yr[i1] = (int16_t)sat16(turn<false, false>(x0, sh[angle], sl[angle], x1, ch[angle], cl[angle]));
          }
        }
        xr += down * a.ldx;
        yr += down * a.ldy;
        angle += down * a.half;
      }
    }
  }
}

}  // namespace

cudaError_t launch_rotary(const int16_t* x, size_t rows, size_t heads, size_t hd, size_t ldx, const nsrl_rotary& rot,
                          const int32_t* positions, size_t seq_len, bool backward, int16_t* y, size_t ldy,
                          cudaStream_t s) {
  if (rows == 0 || heads == 0) return cudaSuccess;
  RotArgs a{};
  a.x = x;
  a.y = y;
  a.ldx = (long long)ldx;
  a.ldy = (long long)ldy;
  a.rows = (long long)rows;
  a.turns = reinterpret_cast<const unsigned long long*>(rot.turns);
  a.positions = positions;
  a.seq_len = (unsigned)std::min<size_t>(std::max<size_t>(seq_len, 1), 0x7fffffff);
  a.heads = (int)heads;
  a.hd = (int)hd;
  a.half = (int)(rot.rotary_dim / 2);
  a.backward = backward;
  a.amplitude = rot.amplitude;
  const bool vec = hd % 16 == 0 && a.half % 8 == 0 && ldx % 8 == 0 && ldy % 8 == 0 &&
                   ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const bool wide = rot.amplitude > (1 << 30);
  // A block is a whole number of rows wide where a row has at most MAX_THREADS
  // items.  It takes ROWS times that many rows, but leaves every SM a block
  // while there are rows for it, and keeps to its angles' shared memory.
  const int unit = vec ? 8 : 1;
  a.turning = a.half / unit;
  a.per_head = a.turning + (x == y ? 0 : ((int)hd - 2 * a.half) / (vec ? 16 : 1));
  a.per_row = a.per_head * a.heads;
  size_t r = std::max<size_t>(1, MAX_THREADS / (size_t)a.per_row);
  size_t wide_rows = r;
  r = std::min(ROWS * r, std::max<size_t>(1, rows / 148));
  r = std::min(r, std::max<size_t>(1, (size_t)MAX_PAIRS / (size_t)a.half));
  wide_rows = std::min(wide_rows, r);
  a.block_rows = (int)r;
  a.down = (int)wide_rows;
  const size_t threads = (std::min<size_t>(MAX_THREADS, wide_rows * (size_t)a.per_row) + 31) / 32 * 32;
  a.step = (int)threads / a.half;
  a.along = (int)threads % a.half;
  auto magic = [](int d) { return ((1u << 22) + (unsigned)d - 1) / (unsigned)d; };
  a.by_row = magic(a.per_row);
  a.by_head = magic(a.per_head);
  a.by_half = magic(a.half);
  const size_t blocks = (rows + r - 1) / r;
  if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
  const double n = (double)rows * (double)heads * (double)hd;
  ProfScope prof("rotary", s, 3.0 * (double)rows * (double)heads * (double)rot.rotary_dim, 4.0 * n);
  auto* kernel = vec ? (rot.interleaved ? (wide ? rotary_kernel<true, true, true> : rotary_kernel<true, true, false>)
                                        : (wide ? rotary_kernel<true, false, true> : rotary_kernel<true, false, false>))
                     : (rot.interleaved ? (wide ? rotary_kernel<false, true, true> : rotary_kernel<false, true, false>)
                                        : (wide ? rotary_kernel<false, false, true> : rotary_kernel<false, false, false>));
  const cudaError_t e = launch_pdl(kernel, dim3((unsigned)blocks), dim3((unsigned)threads), 16 * r * (size_t)a.half, s, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace nsrl
