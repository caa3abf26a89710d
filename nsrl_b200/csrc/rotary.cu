// Rotary positions on int16 rows, forward and backward (nsrl_rotary_rows).
//
// A pair (x0, x1) at position p turns by the angle a = p * turn, kept as a
// 64-bit fraction of a turn, so the product wraps where the angle does and far
// positions keep every bit.  cos and sin come from the nearest of 1,024 points
// of the circle and the remaining angle d (|d| <= 2^-11 turn = 0.0031 rad):
// cos d = 1 - d^2 / 2 within 4e-12, sin d = d within 5e-9, both below 2^-27.
//
// Bound by memory: 2 bytes in and 2 out per element, against about 6 integer
// instructions; the angle work is done once per (row, pair) into shared
// memory and read by every head.  A block takes `rows` rows so that each of
// its 256 threads has about four items (16 dims: two 16-byte loads and
// stores) per head sweep, and asks for its first four items before it works
// out the angles, which hides that work behind the loads.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace nsrl {
namespace {

__device__ const int32_t d_quarter_lut[257] = {NSRL_QUARTER_LUT_VALUES};

constexpr int THREADS = 256;
constexpr int MAX_PAIRS = 2048;  // (row, pair) angles of a block: 16 KB of shared memory
constexpr int ITEMS = 4;         // items a thread loads ahead

struct RotArgs {
  const int16_t* x;
  int16_t* y;
  long long ldx, ldy, rows;
  const unsigned long long* turns;
  const int32_t* positions;
  unsigned seq_len;
  int heads, hd, half, backward, amplitude;
  int block_rows;
};

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
  c = C0 - (int)(((long long)C0 * h256 + (long long)S0 * r + half) >> 38);
  s = S0 - (int)(((long long)S0 * h256 - (long long)C0 * r + half) >> 38);
  if (amplitude != (1 << 30)) {
    // |c| may pass 2^30 by one, so an amplitude near 2 may reach 2^31: held to 2^31 - 1
    c = (int)max(-2147483647ll, min(2147483647ll, ((long long)c * amplitude + (1ll << 29)) >> 30));
    s = (int)max(-2147483647ll, min(2147483647ll, ((long long)s * amplitude + (1ll << 29)) >> 30));
  }
}

// rhu(x0 * c + x1 * s, 30), not yet saturated; the sum stays below 2^48.
__device__ __forceinline__ int turn(int x0, int c, int x1, int s) {
  const long long t = (long long)x0 * c + ((long long)x1 * s + (1ll << 29));
  return (int)(t >> 30);
}

// VEC: an item is 16 dims of a head (8 pairs, or 16 dims past rotary_dim),
// two 16-byte accesses.  Otherwise an item is one pair, or one dim past rotary_dim.
template <bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const RotArgs a) {
  extern __shared__ __align__(16) int32_t angles[];  // c [rows][half], then s
  int32_t* const sc = angles;
  int32_t* const ss = angles + a.block_rows * a.half;
  const long long row0 = (long long)blockIdx.x * a.block_rows;
  const int rows = (int)min((long long)a.block_rows, a.rows - row0);
  // items of a head: the pairs, then (out of place only) the dims that pass through
  const int turning = VEC ? a.half / 8 : a.half;
  const int passing = a.x == a.y ? 0 : (VEC ? (a.hd - 2 * a.half) / 16 : a.hd - 2 * a.half);
  const int per_head = turning + passing, per_row = per_head * a.heads;
  const int items = rows * per_row;

  // An item's place, stepped from one to the next by THREADS in mixed radix:
  // two divisions a thread instead of two an item.
  struct Place {
    int row, head, slot;
  };
  const int step_row = THREADS / per_row, step_head = THREADS % per_row / per_head, step_slot = THREADS % per_head;
  auto next = [&](Place& p) {
    p.slot += step_slot;
    p.head += step_head;
    p.row += step_row;
    if (p.slot >= per_head) {
      p.slot -= per_head;
      ++p.head;
    }
    if (p.head >= a.heads) {
      p.head -= a.heads;
      ++p.row;
    }
  };
  // element offsets of an item's two accesses within its row, and its first pair (-1: passes through)
  auto offsets = [&](const Place& p, int& i0, int& i1) -> int {
    const int base = p.head * a.hd;
    if (p.slot < turning) {
      const int pair = VEC ? 8 * p.slot : p.slot;
      i0 = base + (INTERLEAVED ? 2 * pair : pair);
      i1 = INTERLEAVED ? i0 + (VEC ? 8 : 1) : i0 + a.half;
      return pair;
    }
    i0 = base + 2 * a.half + (VEC ? 16 : 1) * (p.slot - turning);
    i1 = i0 + (VEC ? 8 : 0);
    return -1;
  };

  griddep_wait();
  griddep_launch();
  uint4 v0[ITEMS], v1[ITEMS];
  auto load = [&](const Place& p, uint4& u0, uint4& u1) {
    int i0, i1;
    offsets(p, i0, i1);
    const int16_t* x = a.x + (row0 + p.row) * a.ldx;
    if (VEC) {
      u0 = *reinterpret_cast<const uint4*>(x + i0);
      u1 = *reinterpret_cast<const uint4*>(x + i1);
    } else {
      u0.x = (uint32_t)(uint16_t)x[i0];
      u1.x = (uint32_t)(uint16_t)x[i1];
    }
  };
  Place start;
  start.row = threadIdx.x / per_row;
  start.head = threadIdx.x % per_row / per_head;
  start.slot = threadIdx.x % per_head;
  Place at = start;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    if (threadIdx.x + k * THREADS < items) load(at, v0[k], v1[k]);
    next(at);
  }
  {
    int row = threadIdx.x / a.half, pair = threadIdx.x % a.half;
    const int down = THREADS / a.half, along = THREADS % a.half;
    for (int i = threadIdx.x; i < rows * a.half; i += THREADS) {
      const long long r = row0 + row;
      const long long p = a.positions ? (long long)a.positions[r] : (long long)((unsigned)r % a.seq_len);
      int c, s;
      cos_sin_q30((unsigned long long)p * a.turns[pair], a.amplitude, c, s);
      sc[i] = c;
      ss[i] = a.backward ? -s : s;
      row += down;
      pair += along;
      if (pair >= a.half) {
        pair -= a.half;
        ++row;
      }
    }
  }
  __syncthreads();

  at = start;
  for (int it0 = threadIdx.x; it0 < items; it0 += ITEMS * THREADS) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const Place here = at;
      next(at);
      if (it0 + k * THREADS >= items) continue;
      if (it0 >= ITEMS * THREADS) load(here, v0[k], v1[k]);  // past the items loaded ahead
      int i0, i1;
      const int pair = offsets(here, i0, i1);
      int16_t* p = a.y + (row0 + here.row) * a.ldy;
      const int32_t* c = sc + here.row * a.half + pair;
      const int32_t* s = ss + here.row * a.half + pair;
      if (VEC) {
        uint4 o0 = v0[k], o1 = v1[k];
        if (pair >= 0) {
          int cw[8], sw[8], r0[8], r1[8];
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            *reinterpret_cast<int4*>(cw + i) = *reinterpret_cast<const int4*>(c + i);
            *reinterpret_cast<int4*>(sw + i) = *reinterpret_cast<const int4*>(s + i);
          }
          int e[16];
          unpack8(v0[k], *reinterpret_cast<int(*)[8]>(e));
          unpack8(v1[k], *reinterpret_cast<int(*)[8]>(e + 8));
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int x0 = e[INTERLEAVED ? 2 * i : i], x1 = e[INTERLEAVED ? 2 * i + 1 : 8 + i];
            r0[i] = turn(x0, cw[i], x1, -sw[i]);
            r1[i] = turn(x0, sw[i], x1, cw[i]);
          }
          if (INTERLEAVED) {
            o0 = make_uint4(pack_sat16(r1[0], r0[0]), pack_sat16(r1[1], r0[1]), pack_sat16(r1[2], r0[2]),
                            pack_sat16(r1[3], r0[3]));
            o1 = make_uint4(pack_sat16(r1[4], r0[4]), pack_sat16(r1[5], r0[5]), pack_sat16(r1[6], r0[6]),
                            pack_sat16(r1[7], r0[7]));
          } else {
            o0 = make_uint4(pack_sat16(r0[1], r0[0]), pack_sat16(r0[3], r0[2]), pack_sat16(r0[5], r0[4]),
                            pack_sat16(r0[7], r0[6]));
            o1 = make_uint4(pack_sat16(r1[1], r1[0]), pack_sat16(r1[3], r1[2]), pack_sat16(r1[5], r1[4]),
                            pack_sat16(r1[7], r1[6]));
          }
        }
        *reinterpret_cast<uint4*>(p + i0) = o0;
        *reinterpret_cast<uint4*>(p + i1) = o1;
      } else {
        const int x0 = (int)(int16_t)v0[k].x, x1 = (int)(int16_t)v1[k].x;
        p[i0] = (int16_t)(pair >= 0 ? sat16(turn(x0, c[0], x1, -s[0])) : x0);
        if (pair >= 0) p[i1] = (int16_t)sat16(turn(x0, s[0], x1, c[0]));
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
  // Rows of a block: about ITEMS items a thread, at least one block an SM
  // while there are rows for it, and angles that fit the shared memory.
  const size_t per_row = std::max<size_t>(1, heads * (vec ? hd / 16 : hd - (size_t)a.half));
  size_t r = std::max<size_t>(1, (size_t)(ITEMS * THREADS) / per_row);
  r = std::min(r, std::max<size_t>(1, rows / 148));
  r = std::min(r, std::max<size_t>(1, (size_t)MAX_PAIRS / (size_t)a.half));
  a.block_rows = (int)r;
  const size_t blocks = (rows + r - 1) / r;
  if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
  const double n = (double)rows * (double)heads * (double)hd;
  ProfScope prof("rotary", s, 3.0 * (double)rows * (double)heads * (double)rot.rotary_dim, 4.0 * n);
  auto* kernel = vec ? (rot.interleaved ? rotary_kernel<true, true> : rotary_kernel<true, false>)
                     : (rot.interleaved ? rotary_kernel<false, true> : rotary_kernel<false, false>);
  const cudaError_t e = launch_pdl(kernel, dim3((unsigned)blocks), dim3(THREADS), 8 * r * (size_t)a.half, s, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace nsrl
