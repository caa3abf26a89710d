// Attention of one query per sequence over the 4-bit cache
// (nsrl_attention_decode_q4): the logits, base-2 softmax and context of
// nsrl_attention_decode (attention.cu) on the values the codes stand for.
//
// With value = zero + scale * code per group g of 32 dims,
//   q . k   = sum_g scale_g (sum_i q_i code_i) + zero_g (sum_i q_i)
//   sum p v = sum_j p_j zero_jg + (p_j scale_jg) code_j.
//
// The Q15 weights need the row's maximum and sum before the first value is
// weighed.  Two forms, both of which read the cache once:
//   WHOLE   one launch; a (sequence, head) is one CTA, or a cluster of them
//           where rows are few: each takes a contiguous share of the slots,
//           keeps their logits in shared memory, and the cluster exchanges
//           maximum, sum and partial contexts through distributed shared memory.
//           Many rows of unlike lengths begin with the longest (order_kernel).
//   split   three launches over fixed chunks of slots: KEYS writes logits (4
//           bytes a slot) and each chunk's maximum, sums_kernel each chunk's
//           sum, VALUES each chunk's context; the last chunk of a row to arrive
//           adds them up (integers: in any order the same).  No CTA waits for
//           another, and chunks spread evenly over the SMs.
// plan_of() chooses, by sizes alone.
// Scores go on from call to call, so a call with a bad length, or whose status
// already holds a rejection, leaves all of them: it can be mended and made again.
// Bad lengths are known before the first score changes: every CTA looks at all of
// them (fewer than SORT_ROWS, so at most three a thread), or an earlier launch of
// the call has.  A row with a logit outside 32 bits leaves its own.
//
// Bound by memory (80 bytes a slot of 64 dims, 88 with scores) while an SM
// spends less than about 3.5 cycles on a slot, that is some 14 instructions of
// a warp on 32 slots each cycle it has; the integer pipes take one every other
// cycle.  So instructions are counted:
//   keys:   a lane owns a slot and loads its whole row (256 dims: eight lanes
//           a slot, a group each); codes widen to bytes and
//           meet the query's high (signed) and low (unsigned) byte planes in
//           dp4a, 32 a slot.
//   values: int8 MMAs (m16n8k32): A = 16 dims x 32 slots (transposing matrix
//           loads from a kilobyte that the warp has to itself, and a PRMT), B =
//           the four byte planes of p_j scale_jg of two groups, one column each.
// Warps work on units of 32 slots by themselves, the next unit's loads under
// way: a ring of bulk copies between warps cost as many instructions in waits
// and index arithmetic as the products themselves (keys of 32 rows of 8,192
// slots: 174 instructions a unit and 18 us even without the loads).
// Everything is exact in s32 until it is combined in 64 bits.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace cg = cooperative_groups;

namespace nsrl {
namespace {

constexpr int MAX_CLUSTER = 16;
constexpr int UNIT = 32;             // slots of a warp's step
constexpr int LENGTHS = 64;          // classes of length
constexpr size_t SORT_ROWS = 592, SORT_BATCH = 4096;  // from so many rows, up to so many sequences: long ones first
constexpr size_t MANY_ROWS = 888, MANY_SLOTS = 10240;  // from so many rows up to so many slots: 8 warps a CTA
constexpr size_t MAX_SHARE = 32768;  // logits of a CTA: 128 KB
constexpr int CHUNK = 2048;          // slots of a CTA of the split form
constexpr int FEW_SLOTS = 2048;      // up to which a CTA of the one-launch form has 8 warps, 16 above
constexpr size_t SPLIT_SLOTS = MAX_CLUSTER * FEW_SLOTS;  // capacity from which few rows take the split form

template <int HD>
struct Q4Shape {
  static constexpr int WORDS = HD / 8;             // code words of a slot
  static constexpr int G = HD < 32 ? 1 : HD / 32;  // groups
  static constexpr int GW = HD < 32 ? HD / 8 : 4;  // code words of a group
  static constexpr int PAIRS = (G + 1) / 2;        // pairs of groups, 64 dims each
  static constexpr int SHIFT = HD == 16 ? 2 : HD == 64 ? 3 : 4;
};

// Flags that a CTA of the running launch may set at any moment: not asked for, so
// that what a call does to the scores does not depend on the order of its CTAs.
constexpr unsigned long long FOUND_LATE = NSRL_FLAG_LOGIT_RANGE | NSRL_FLAG_ALL_MASKED;

struct AttendArgs {
  nsrl_q4_cache c;
  const int16_t* q;
  long long ldq;
  const int32_t* lens;
  int len_offset;
  int16_t* ctx;
  nsrl_device_status* st;
  // WHOLE's scratch
  int2* order;       // [batch]: (sequence, length), the longest first; NULL: as they come
  int length_shift;  // class of a length
  bool lens_known;   // an earlier launch has flagged the bad lengths
  // the split form's scratch
  int chunks;           // of a row of `capacity` slots
  int32_t* logits;      // [batch * heads][capacity]
  int32_t* chunk_max;   // [batch * heads][chunks]
  unsigned* chunk_sum;  // [batch * heads][chunks]
  unsigned* arrived;    // [batch * heads]: chunks whose context is written
  long long* partial;   // [batch * heads][chunks][head_dim]
};

__device__ __forceinline__ unsigned long long flags_of(const AttendArgs& a) {
  return *reinterpret_cast<const volatile unsigned long long*>(&a.st->flags);
}

__device__ __forceinline__ bool bad_length(const AttendArgs& a, long long len) {
  return len <= 0 || len > (long long)a.c.capacity;
}

__device__ __forceinline__ int dp4a_us(uint32_t a, uint32_t b, int c) {  // unsigned x signed bytes
  int d;
  asm("dp4a.u32.s32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ int dp4a_uu(uint32_t a, uint32_t b, int c) {
  int d;
  asm("dp4a.u32.u32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

__device__ __forceinline__ void mma_u8u8(int (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

__device__ __forceinline__ int add_sat(int x, int y) {
  int r;
  asm("add.sat.s32 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}

// Four 8 x 8 matrices of 16-bit elements, transposed; lane l gives the 16-byte row l & 7 of matrix l >> 3.
__device__ __forceinline__ void load_matrices(uint32_t row, uint32_t* w) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(row)
               : "memory");
}

constexpr uint32_t LOW = 0x0F0F0F0Fu, HIGH = 0xF0F0F0F0u;

// Byte t of the words of a quad's four lanes, in lane order (a 4 x 4 byte transpose).
__device__ __forceinline__ uint32_t quad_plane(uint32_t x, int t) {
  x = __byte_perm(x, __shfl_xor_sync(0xffffffffu, x, 2), (t & 2) ? 0x3276 : 0x5410);
  return __byte_perm(x, __shfl_xor_sync(0xffffffffu, x, 1), (t & 1) ? 0x3715 : 0x6240);
}

// Weight of a logit (exp2_neg_q15 of lg - mx <= 0, whose magnitude fits 32 bits).
// From 15 * 256 on it is 0: so is MASKED_LOGIT's, INT_MIN, unless mx is that low.
__device__ __forceinline__ unsigned weight(const int16_t* lut, int lg, int mx) {
  const unsigned mag = min((unsigned)mx - (unsigned)lg, 15u * 256u);
  return (unsigned)lut[mag & 255] >> (mag >> 8);
}

// recip_sum_q31 with the table in shared memory.  Where any logit counts, the
// slot at the maximum weighs 32767, so the sum is at least that, the result at most
// 65793.  A smaller one can only come from a workspace that another call writes to
// at the same time: a wrong answer then, but no access outside the table.
__device__ __forceinline__ unsigned reciprocal(const uint32_t* recip, unsigned long long sum) {
  if (sum < 32767) return 0;
  const int shift = 63 - __clzll((long long)sum) - 7;
  return recip[((unsigned)(sum >> shift) & 255u) - 128] >> shift;
}

// The sum of weight() over n logits at `logits` (16-byte aligned), this thread's part.
template <int THREADS>
__device__ __forceinline__ unsigned weigh(const int16_t* lut, const int32_t* logits, int n, int mx) {
  unsigned sum = 0;
  const bool low = mx < INT_MIN + 15 * 256;  // MASKED_LOGIT would gather weight
  const int none = (int)((unsigned)mx - 15u * 256u);
#pragma unroll 2
  for (int j = 4 * (int)threadIdx.x; j < n; j += 4 * THREADS) {
    int4 lg = *reinterpret_cast<const int4*>(logits + j);
    if (j + 3 >= n || low) {
      if (lg.x == INT_MIN) lg.x = none;
      if (lg.y == INT_MIN || j + 1 >= n) lg.y = none;
      if (lg.z == INT_MIN || j + 2 >= n) lg.z = none;
      if (lg.w == INT_MIN || j + 3 >= n) lg.w = none;
    }
    sum += weight(lut, lg.x, mx) + weight(lut, lg.y, mx) + weight(lut, lg.z, mx) + weight(lut, lg.w, mx);
  }
  return sum;
}

// ---------------------------------------------------------------------- keys
// The query of one (sequence, head) in shared memory: per group and code word
// {h of the even dims, h of the odd dims, l even, l odd} with q = 256 h + l, then
// 16 times the group's sum of q.
template <int HD>
struct Query {
  uint4 word[Q4Shape<HD>::WORDS];
  int sum16[Q4Shape<HD>::G];
};

// Warp 0 lays it out; the caller synchronises.
template <int HD>
__device__ __forceinline__ void lay_out(Query<HD>& q, const int16_t* row) {
  using S = Q4Shape<HD>;
  const int lane = threadIdx.x;
  if (lane >= S::WORDS) return;
  uint32_t w[4] = {0, 0, 0, 0};
  int sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int v = row[8 * lane + i];
    sum += v;
    w[i & 1] |= (uint32_t)((v >> 8) & 255) << (8 * (i >> 1));
    w[2 + (i & 1)] |= (uint32_t)(v & 255) << (8 * (i >> 1));
  }
  constexpr unsigned mask = S::WORDS >= 32 ? 0xffffffffu : (1u << S::WORDS) - 1;
#pragma unroll
  for (int o = 1; o < S::GW; o <<= 1) sum += __shfl_xor_sync(mask, sum, o);
  q.word[lane] = make_uint4(w[0], w[1], w[2], w[3]);
  if (lane % S::GW == 0) q.sum16[lane / S::GW] = 16 * sum;
}

// A slot's row of codes and scales.
template <int HD>
struct KeyRow {
  uint32_t code[Q4Shape<HD>::WORDS];
  uint32_t scale[Q4Shape<HD>::G];

  __device__ __forceinline__ void load(const nsrl_q4_cache& c, size_t slot) {
    const uint8_t* p = c.k_codes + slot * (HD / 2);
    const uint32_t* s = c.k_scales + slot * Q4Shape<HD>::G;
    if constexpr (HD == 16) {
      const uint2 x = __ldcs(reinterpret_cast<const uint2*>(p));
      code[0] = x.x, code[1] = x.y;
      scale[0] = __ldcs(s);
    } else {
#pragma unroll
      for (int i = 0; i < Q4Shape<HD>::WORDS; i += 4) {
        const uint4 x = __ldcs(reinterpret_cast<const uint4*>(p) + i / 4);
        code[i] = x.x, code[i + 1] = x.y, code[i + 2] = x.z, code[i + 3] = x.w;
      }
#pragma unroll
      for (int i = 0; i < Q4Shape<HD>::G; i += 2) {
        const uint2 x = __ldcs(reinterpret_cast<const uint2*>(s) + i / 2);
        scale[i] = x.x, scale[i + 1] = x.y;
      }
    }
  }
};

// 16 q . k of R slots (odd dims stay in the high half bytes, the even ones
// catch up); the query's words are read once for all of them.
template <int HD, int R>
__device__ __forceinline__ void dots16(const Query<HD>& query, const KeyRow<HD> (&row)[R], long long (&v)[R]) {
  using S = Q4Shape<HD>;
#pragma unroll
  for (int r = 0; r < R; ++r) v[r] = 0;
#pragma unroll
  for (int g = 0; g < S::G; ++g) {
    int he[R], ho[R], le[R], lo[R];
#pragma unroll
    for (int r = 0; r < R; ++r) he[r] = ho[r] = le[r] = lo[r] = 0;
#pragma unroll
    for (int k = 0; k < S::GW; ++k) {
      const uint4 q = query.word[S::GW * g + k];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t w = row[r].code[S::GW * g + k];
        he[r] = dp4a_us(w & LOW, q.x, he[r]);
        ho[r] = dp4a_us(w & HIGH, q.y, ho[r]);
        le[r] = dp4a_uu(w & LOW, q.z, le[r]);
        lo[r] = dp4a_uu(w & HIGH, q.w, lo[r]);
      }
    }
    const int sum16 = query.sum16[g];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int dot = (he[r] * 256 + le[r]) * 16 + (ho[r] * 256 + lo[r]);  // 16 sum q code, below 2^28
      v[r] += (long long)dot * (int)(row[r].scale[g] & 0xFFFF) + (long long)sum16 * ((int)row[r].scale[g] >> 16);
    }
  }
}

// A unit of 256-dim rows: eight lanes a row, each one group of it, so that a load
// of the warp takes four whole rows and the query stays in registers.  Step i of a
// lane is row 4 i + (lane >> 3).  64 rows of 8,192 take 50 us, and 60 with a lane a
// row; at 64 dims the same with two lanes a row is slower (35.2 for 34.3 us, 256
// rows of 8,192): its registers pass the 64 that two CTAs of 16 warps leave
// (the kept form is at that limit itself and spills 76 bytes).
struct KeyUnit256 {
  uint4 code[8];
  uint32_t scale[8];

  template <bool ALL>
  __device__ __forceinline__ void load(const nsrl_q4_cache& c, size_t slot, int left) {
    const int lane = threadIdx.x & 31, r = lane >> 3;
    const uint4* p = reinterpret_cast<const uint4*>(c.k_codes + slot * 128) + lane;
    const uint32_t* s = c.k_scales + slot * 8 + lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool there = ALL || 4 * i + r < left;
      code[i] = there ? __ldcs(p + 32 * i) : make_uint4(0, 0, 0, 0);
      scale[i] = there ? __ldcs(s + 32 * i) : 0u;
    }
  }

  // 16 q . k of row 4 (lane & 7) + (lane >> 3); q: this lane's group of the query
  __device__ __forceinline__ long long dot16(const uint4 (&q)[4], int sum16) const {
    const int g = threadIdx.x & 7;
    long long v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
      int he = 0, ho = 0, le = 0, lo = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        he = dp4a_us(w[k] & LOW, q[k].x, he);
        ho = dp4a_us(w[k] & HIGH, q[k].y, ho);
        le = dp4a_uu(w[k] & LOW, q[k].z, le);
        lo = dp4a_uu(w[k] & HIGH, q[k].w, lo);
      }
      const int dot = (he * 256 + le) * 16 + (ho * 256 + lo);
      v[i] = (long long)dot * (int)(scale[i] & 0xFFFF) + (long long)sum16 * ((int)scale[i] >> 16);
    }
    // the eight lanes' groups add up, and lane g keeps step g
#pragma unroll
    for (int o = 4; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < o; ++i) {
        const bool upper = g & o;
        const long long give = upper ? v[i] : v[i + o];
        v[i] = (upper ? v[i + o] : v[i]) + __shfl_xor_sync(0xffffffffu, give, o);
      }
    return v[0];
  }
};

// Logits of n slots from slot0; returns this warp's maximum (INT_MIN: none
// counts; MASKED_LOGIT is INT_MIN and never raises it).  A step takes two whole
// units (one at 256 dims) with the next step's rows under way; what is left over
// goes unit by unit.
// `ready` is called once, after the first loads and before the query is read,
// `outside` by a lane that had a logit outside 32 bits.
template <int HD, int WARPS, typename Ready, typename Outside>
__device__ __forceinline__ int keys_pass(const AttendArgs& a, const Query<HD>& query, size_t slot0, int n,
                                         int32_t* logits, Ready ready, Outside outside) {
  using S = Q4Shape<HD>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int mx = INT_MIN;
  bool bad = false;
  auto put = [&](int j, long long v) {
    const long long lg = v >> (S::SHIFT + 4);
    bad = bad || lg != (long long)(int)lg;
    logits[j] = (int)lg;
    mx = max(mx, (int)lg);
  };
  const int whole = n / UNIT;
  int u = warp;
  if constexpr (HD != 256) {
    KeyRow<HD> row[2], next[2];
    bool two = u + WARPS < whole;
    if (two) {
      next[0].load(a.c, slot0 + u * UNIT + lane);
      next[1].load(a.c, slot0 + (u + WARPS) * UNIT + lane);
    }
    ready();
    while (two) {
      row[0] = next[0];
      row[1] = next[1];
      const int at = u * UNIT + lane;
      u += 2 * WARPS;
      two = u + WARPS < whole;
      if (two) {
        next[0].load(a.c, slot0 + u * UNIT + lane);
        next[1].load(a.c, slot0 + (u + WARPS) * UNIT + lane);
      }
      long long v[2];
      dots16<HD, 2>(query, row, v);
      put(at, v[0]);
      put(at + WARPS * UNIT, v[1]);
    }
    for (; u * UNIT < n; u += WARPS) {
      const int j = u * UNIT + lane;
      if (j >= n) continue;
      KeyRow<HD> row[1];
      row[0].load(a.c, slot0 + j);
      long long v[1];
      dots16<HD, 1>(query, row, v);
      put(j, v[0]);
    }
  } else {
    KeyUnit256 unit, next;
    if (u < whole) next.load<true>(a.c, slot0 + u * UNIT, UNIT);
    ready();
    const int g = lane & 7, mine = 4 * g + (lane >> 3);
    const uint4 q[4] = {query.word[4 * g], query.word[4 * g + 1], query.word[4 * g + 2], query.word[4 * g + 3]};
    const int sum16 = query.sum16[g];
    while (u < whole) {
      unit = next;
      const int at = u * UNIT + mine;
      u += WARPS;
      if (u < whole) next.load<true>(a.c, slot0 + u * UNIT, UNIT);
      put(at, unit.dot16(q, sum16));
    }
    if (u == whole && n % UNIT != 0) {
      unit.load<false>(a.c, slot0 + u * UNIT, n % UNIT);
      const long long v = unit.dot16(q, sum16);
      if (mine < n % UNIT) put(u * UNIT + mine, v);
    }
  }
  if (bad) {
    nsrl_flag(a.st, NSRL_FLAG_LOGIT_RANGE);
    outside();
  }
  return __reduce_max_sync(0xffffffffu, mx);
}

// -------------------------------------------------------------------- values
// A warp's unit is 32 slots of one pair of groups (64 dims).  Transposing
// matrix loads give lane (g, t) bytes 2 g and 2 g + 1 of a group's row for
// slots 8 m + 2 t and 8 m + 2 t + 1; two of them and a PRMT make one byte of
// four slots.  16 dims a head (8-byte rows): byte g of slots 4 j + t from words.
// A byte holds an even and an odd dim: row g of its MMA takes the byte as it is
// (even + 16 odd), row g + 8 its high half (16 odd), and they part at the end.
// Slot `own` is this lane's to weigh (p, its score, p scale); the byte planes of
// p scale then go to the lanes of their column.
template <int HD>
struct ValueUnit {
  uint4 code[2];  // HD 16: the first 8 bytes
  uint2 scale;
  int logit, score;
};

// This lane's places in a row's (or chunk's) first unit; a unit further on they
// move by constants.  FAR: the logits are in global memory and come with the
// rows; otherwise they are read from shared memory when they are due.
template <int HD, bool FAR>
struct ValuePlaces {
  using S = Q4Shape<HD>;
  const uint8_t* code;
  const uint32_t* scale;
  const int32_t* logit;
  int32_t* score;  // NULL: no scores, or another warp's to keep
  int own, pair;

  __device__ __forceinline__ ValuePlaces(const AttendArgs& a, size_t slot0, const int32_t* logits) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    pair = warp % S::PAIRS;
    // The quad's slots are those of k = 4 (g & 3) + 16 (g >> 2) and the three after it.
    own = 16 * (g >> 2) + (HD == 16 ? 4 * t + (g & 3) : 8 * (t >> 1) + 2 * (g & 3) + (t & 1));
    code = HD == 16 ? a.c.v_codes + (slot0 + lane) * (HD / 2)
                    : a.c.v_codes + (slot0 + (lane >> 1)) * (HD / 2) + 32 * pair + 16 * (lane & 1);
    scale = a.c.v_scales + (slot0 + own) * S::G + (HD == 16 ? 0 : 2 * pair);
    logit = logits + own;
    score = a.c.scores && pair == 0 ? a.c.scores + slot0 + own : nullptr;
  }

  // ALL: every slot of the unit is there; otherwise `left` of them are
  template <bool ALL>
  __device__ __forceinline__ void load(ValueUnit<HD>& u, int unit, int left) const {
    const int lane = threadIdx.x & 31;
    // rows past the end are inside the capacity up to the next multiple of 16 slots
    const int last = (left + 15) & ~15;
    const uint8_t* c = code + (size_t)(unsigned)unit * (UNIT * HD / 2);
    if constexpr (HD == 16) {
      const uint2 x = ALL || lane < last ? __ldcs(reinterpret_cast<const uint2*>(c)) : make_uint2(0, 0);
      u.code[0].x = x.x, u.code[0].y = x.y;
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        u.code[e] = ALL || 16 * e + (lane >> 1) < last ? __ldcs(reinterpret_cast<const uint4*>(c + e * 16 * (HD / 2)))
                                                         : make_uint4(0, 0, 0, 0);
    }
    const bool mine = ALL || own < left;
    const uint32_t* s = scale + (size_t)(unsigned)unit * (UNIT * S::G);
    if constexpr (HD == 16)
      u.scale = make_uint2(mine ? __ldcs(s) : 0u, 0u);
    else
      u.scale = mine ? __ldcs(reinterpret_cast<const uint2*>(s)) : make_uint2(0, 0);
    if (FAR) u.logit = mine ? logit[unit * UNIT] : INT_MIN;
    u.score = score && mine ? score[unit * UNIT] : 0;
  }
};

// The first unit of this warp, asked for ahead of values_pass.
template <int HD, int WARPS, bool FAR>
__device__ __forceinline__ void first_values(const ValuePlaces<HD, FAR>& at, int n, ValueUnit<HD>& next) {
  const int u = (int)(threadIdx.x >> 5) / Q4Shape<HD>::PAIRS;
  if ((u + 1) * UNIT <= n) at.template load<true>(next, u, UNIT);
}

// Context of n slots into part[HD] (this warp's row; only the pair's dims are written).
template <int HD, int WARPS, bool FAR>
__device__ __forceinline__ void values_pass(const ValuePlaces<HD, FAR>& at, ValueUnit<HD> next, int n,
                                            const int16_t* lut, int mx, unsigned inv, uint8_t* buffer,
                                            long long* part) {
  using S = Q4Shape<HD>;
  constexpr int MMAS = HD == 16 ? 1 : 4;
  constexpr int STEP = WARPS / S::PAIRS;  // units from one of this warp's to its next
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int pair = at.pair, own = at.own;
  int acc[MMAS][4];
#pragma unroll
  for (int i = 0; i < MMAS; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0;
  long long zero_part[2] = {0, 0};  // sum of p zero over this lane's slots, per group of the pair
  const int from = 4 * t + (g & 3);  // the lane with plane g & 3 of the slots of k = 4 t; 16 further, of 16 + 4 t
  const uint32_t byte2 = (uint32_t)(g & 3) | ((uint32_t)((g & 3) + 4) << 4);  // byte g & 3 of two words
  // Rows of 32 bytes in the warp's buffer, the halves of rows 4 .. 7 of eight
  // swapped so that the matrix loads' eight rows meet no bank twice.
  const uint32_t store_at = smem_u32(buffer) + 32 * (lane >> 1) + 16 * ((lane & 1) ^ ((lane >> 3) & 1));
  const uint32_t load_at = smem_u32(buffer) + 32 * lane + 16 * ((lane >> 2) & 1);
  auto add = [&](const ValueUnit<HD>& unit, int logit, int32_t* score) {  // score: NULL, or this lane's slot's
    const int p = logit == INT_MIN ? 0 : (int)min((weight(lut, logit, mx) * inv + 32768u) >> 16, 32767u);
    if (score) *score = add_sat(unit.score, p);
    uint32_t w[8];
    if constexpr (HD == 16) {
      *reinterpret_cast<uint2*>(buffer + 8 * lane) = make_uint2(unit.code[0].x, unit.code[0].y);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = *reinterpret_cast<const uint32_t*>(buffer + 8 * (4 * j + t) + 4 * (g >> 2));
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(store_at + 512 * e), "r"(unit.code[e].x),
                     "r"(unit.code[e].y), "r"(unit.code[e].z), "r"(unit.code[e].w)
                     : "memory");
      __syncwarp();
      load_matrices(load_at, w);           // w[4 e + m]: group e of slots 8 m ..
      load_matrices(load_at ^ 16, w + 4);
    }
    __syncwarp();
    uint32_t bf[2];
    zero_part[0] += (long long)p * ((int)unit.scale.x >> 16);
    const uint32_t plane0 = quad_plane((uint32_t)p * (unit.scale.x & 0xFFFF), t);
    if constexpr (HD == 16) {
      bf[0] = __shfl_sync(0xffffffffu, plane0, from);
      bf[1] = __shfl_sync(0xffffffffu, plane0, from + 16);
    } else {
      zero_part[1] += (long long)p * ((int)unit.scale.y >> 16);
      const uint32_t plane1 = quad_plane((uint32_t)p * (unit.scale.y & 0xFFFF), t);
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const uint32_t x = __shfl_sync(0xffffffffu, plane0, from + 16 * o);
        const uint32_t y = __shfl_sync(0xffffffffu, plane1, from + 16 * o);
        bf[o] = (g >> 2) ? y : x;
      }
    }
#pragma unroll
    for (int i = 0; i < MMAS; ++i) {
      uint32_t x, y;  // the byte of k = 4 t .. and of k = 16 + 4 t ..
      if constexpr (HD == 16) {
        x = __byte_perm(__byte_perm(w[0], w[1], byte2), __byte_perm(w[2], w[3], byte2), 0x5410);
        y = __byte_perm(__byte_perm(w[4], w[5], byte2), __byte_perm(w[6], w[7], byte2), 0x5410);
      } else {  // MMA i: byte i & 1 of group i >> 1
        const uint32_t* m = w + 4 * (i >> 1);
        x = __byte_perm(m[0], m[1], (i & 1) ? 0x7531 : 0x6420);
        y = __byte_perm(m[2], m[3], (i & 1) ? 0x7531 : 0x6420);
      }
      const uint32_t frag[4] = {x, x & HIGH, y, y & HIGH};
      mma_u8u8(acc[i], frag, bf);
    }
  };
  const int whole = n / UNIT;
  int u = warp / S::PAIRS;
  ValueUnit<HD> unit;
  while (u < whole) {
    unit = next;
    const int here = u * UNIT;
    u += STEP;
    if (u < whole) at.template load<true>(next, u, UNIT);
    add(unit, FAR ? unit.logit : at.logit[here], at.score ? at.score + here : nullptr);
  }
  if (u == whole && n % UNIT != 0) {
    const int left = n % UNIT;
    at.template load<false>(unit, u, left);
    const bool mine = own < left;
    add(unit, !mine ? INT_MIN : FAR ? unit.logit : at.logit[u * UNIT], mine && at.score ? at.score + u * UNIT : nullptr);
  }
  // Columns 2 t and 2 t + 1 are planes 2 (t & 1) and 2 (t & 1) + 1 of group t >> 1
  // of the pair.  s32 is enough: 255 * 255 a slot over at most 8,192 slots a warp.
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    zero_part[0] += __shfl_xor_sync(0xffffffffu, zero_part[0], o);
    if (HD != 16) zero_part[1] += __shfl_xor_sync(0xffffffffu, zero_part[1], o);
  }
#pragma unroll
  for (int i = 0; i < MMAS; ++i)
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const int p0 = o ? acc[i][2] >> 4 : acc[i][0] - acc[i][2], p1 = o ? acc[i][3] >> 4 : acc[i][1] - acc[i][3];
      long long v = ((long long)p0 + ((long long)p1 << 8)) << (16 * (t & 1));
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      const int dim = HD == 16 ? 2 * g + o : 64 * pair + 32 * (i >> 1) + 4 * g + 2 * (i & 1) + o;
      if (t == 2 * (i >> 1)) part[dim] = v + zero_part[i >> 1];
    }
}

// --------------------------------------------------------------- one launch
// Gives `value` to entry `part` of every CTA of the cluster; all of them are
// here once the cluster has synchronised.
template <typename T>
__device__ __forceinline__ void share_out(const cg::cluster_group& cluster, T* values, T value, int part, int parts) {
  if ((int)threadIdx.x < parts) cluster.map_shared_rank(values, threadIdx.x)[part] = value;
  cluster.sync();
}

// The sequences by class of length, the longest first, so that the call does not
// end on a long one that began late.  Within a class in any order: a row's
// results do not depend on when it runs.
__global__ void __launch_bounds__(1024) q4_order_kernel(const AttendArgs a) {
  __shared__ int count[LENGTHS], next[LENGTHS];
  const int tid = threadIdx.x, batch = (int)a.c.batch;
  if (tid < LENGTHS) count[tid] = 0;
  griddep_wait();
  griddep_launch();
  __syncthreads();
  auto length = [&](int i) { return (int)min((long long)a.lens[i] + a.len_offset, (long long)INT_MAX); };
  auto length_class = [&](int len) { return min(max(len, 0) >> a.length_shift, LENGTHS - 1); };
  for (int i = tid; i < batch; i += 1024) {
    const int len = length(i);
    if (bad_length(a, len)) nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
    atomicAdd(&count[length_class(len)], 1);
  }
  __syncthreads();
  if (tid < LENGTHS) {
    int longer = 0;
    for (int k = tid + 1; k < LENGTHS; ++k) longer += count[k];
    next[tid] = longer;
  }
  __syncthreads();
  for (int i = tid; i < batch; i += 1024) {
    const int len = length(i);
    a.order[atomicAdd(&next[length_class(len)], 1)] = make_int2(i, len);
  }
}

// Flags the bad lengths before the attention begins, where a CTA would have too
// many of them to look through.
__global__ void __launch_bounds__(256) q4_screen_kernel(const AttendArgs a) {
  griddep_wait();
  griddep_launch();
  const unsigned b = blockIdx.x * 256 + threadIdx.x;
  if (b < (unsigned)a.c.batch && bad_length(a, (long long)a.lens[b] + a.len_offset))
    nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
}

template <int HD, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, HD == 256 ? 16 / WARPS : 32 / WARPS) attend_q4_kernel(const AttendArgs a) {
  using S = Q4Shape<HD>;
  constexpr int THREADS = 32 * WARPS;
  extern __shared__ __align__(16) int32_t logits[];
  __shared__ Query<HD> query;
  __shared__ __align__(128) uint8_t buffer[WARPS][1024];
  __shared__ int16_t lut[256];
  __shared__ uint32_t recip[128];
  __shared__ int s_max[MAX_CLUSTER], s_redi[WARPS];
  __shared__ unsigned s_red[WARPS];
  __shared__ unsigned long long s_sum[MAX_CLUSTER];
  __shared__ long long s_part[WARPS / S::PAIRS][HD], s_ctx[HD];
  __shared__ int s_hold;  // the scores stay as they are
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 256) lut[tid] = d_exp2_lut[tid];
  if (tid < 128) recip[tid] = d_recip_lut[tid];
  if (tid == 0) s_hold = 0;
  griddep_wait();
  griddep_launch();
  unsigned bh = blockIdx.x / (unsigned)parts, b = bh / (unsigned)a.c.heads;
  const unsigned h = bh - b * (unsigned)a.c.heads;
  long long len;
  if (a.order) {
    const int2 o = a.order[b];
    b = (unsigned)o.x;
    bh = b * (unsigned)a.c.heads + h;
    len = o.y;
  } else {
    len = (long long)a.lens[b] + a.len_offset;
  }
  if (warp == 0) lay_out<HD>(query, a.q + b * a.ldq + (long long)h * HD);
  // The last thread asks for the flags, the others for a length each; they are
  // looked at once the first keys are on their way.  Waiting ahead of the keys cost
  // 5 to 13% of a call, waiting after them 2 to 8%, here 0.2 to 0.4 us in one wave.
  const bool look = a.c.scores && (tid == THREADS - 1 || (!a.lens_known && tid < (int)a.c.batch));
  int said = 0;
  if (look) said = tid == THREADS - 1 ? (int)flags_of(a) : a.lens[tid];
  if (bad_length(a, len)) {  // the same for the whole cluster
    if (tid == 0) nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
    return;
  }
  const int share = ((int)((len + parts - 1) / parts) + UNIT - 1) / UNIT * UNIT;
  const long long first = (long long)part * share;
  const int n = (int)max(0ll, min((long long)share, len - first));
  const size_t slot0 = (size_t)bh * a.c.capacity + (size_t)first;
  int mx = keys_pass<HD, WARPS>(a, query, slot0, n, logits, [&] {
    if (parts > 1)
      cluster.sync();  // every CTA has started: its shared memory may be written
    else
      __syncthreads();
    if (look) {
      bool hold = tid == THREADS - 1 ? (said & ~(int)FOUND_LATE) != 0 : bad_length(a, (long long)said + a.len_offset);
      if (!a.lens_known)
        for (unsigned i = tid + THREADS - 1; i < (unsigned)a.c.batch; i += THREADS - 1)
          hold |= bad_length(a, (long long)a.lens[i] + a.len_offset);
      if (hold) s_hold = 1;
    }
  }, [&] { s_hold = 1; });  // the weights of this row are of no use
  const ValuePlaces<HD, false> at(a, slot0, logits);
  ValueUnit<HD> next;
  first_values<HD, WARPS>(at, n, next);  // under way while the softmax is worked out
  if (lane == 0) s_redi[warp] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) mx = max(mx, s_redi[w]);
  if (parts > 1) {
    share_out(cluster, s_max, mx, part, parts);
    for (int r = 0; r < parts; ++r) mx = max(mx, s_max[r]);
  }
  if (mx == INT_MIN && tid == 0 && part == 0) nsrl_flag(a.st, NSRL_FLAG_ALL_MASKED);
  // Only the sum: the value pass weighs each slot again.  A CTA's sum is at most 2^15 * MAX_SHARE = 2^30.
  const unsigned mine = __reduce_add_sync(0xffffffffu, weigh<THREADS>(lut, logits, n, mx));
  if (lane == 0) s_red[warp] = mine;
  __syncthreads();
  unsigned long long sum = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) sum += s_red[w];
  bool hold = s_hold != 0;
  if (parts > 1) {
    constexpr unsigned long long HELD = 1ull << 40;  // above any sum: 2^30 a CTA
    share_out(cluster, s_sum, sum + (hold ? HELD : 0), part, parts);
    sum = 0;
    for (int r = 0; r < parts; ++r) sum += s_sum[r];
    hold = sum >= HELD;
    sum &= HELD - 1;
  }
  const unsigned inv = mx == INT_MIN ? 0u : reciprocal(recip, sum);
  if (hold) {  // its own copy of the pass: a pointer that may be NULL late costs the other 6% in registers
    ValuePlaces<HD, false> still = at;
    still.score = nullptr;
    values_pass<HD, WARPS>(still, next, n, lut, mx, inv, buffer[warp], s_part[warp / S::PAIRS]);
  } else {
    values_pass<HD, WARPS>(at, next, n, lut, mx, inv, buffer[warp], s_part[warp / S::PAIRS]);
  }
  __syncthreads();
  long long total = 0;
  if (tid < HD) {
#pragma unroll
    for (int w = 0; w < WARPS / S::PAIRS; ++w) total += s_part[w][tid];
  }
  if (parts > 1) {
    if (tid < HD) s_ctx[tid] = total;
    cluster.sync();
    if (part == 0 && tid < HD)
      for (int r = 1; r < parts; ++r) total += cluster.map_shared_rank(s_ctx, r)[tid];
  }
  if (part == 0 && tid < HD)
    a.ctx[b * (long long)(a.c.heads * HD) + (long long)h * HD + tid] = sat_i16(rhu64(total, 15));
  if (parts > 1) cluster.sync();  // no CTA leaves while rank 0 reads its partial context
}

// ------------------------------------------------------------ three launches
// Grids are (batch * heads, chunks): a CTA is one chunk of one row.
constexpr int SPLIT_WARPS = 8, SPLIT_THREADS = 32 * SPLIT_WARPS;

// A chunk's place: false past the row's end (or for a bad length, which KEYS flags).
struct Chunk {
  unsigned bh, b, h;
  int n, live;  // slots; chunks of the row
  size_t slot0;
  long long len;

  __device__ __forceinline__ bool find(const AttendArgs& a) {
    bh = blockIdx.x;
    b = bh / (unsigned)a.c.heads;
    h = bh - b * (unsigned)a.c.heads;
    len = (long long)a.lens[b] + a.len_offset;
    if (bad_length(a, len)) return false;
    const long long first = (long long)blockIdx.y * CHUNK;
    if (first >= len) return false;
    n = (int)min((long long)CHUNK, len - first);
    live = (int)((len + CHUNK - 1) / CHUNK);
    slot0 = (size_t)bh * a.c.capacity + (size_t)first;
    return true;
  }
};

template <int HD>
__global__ void __launch_bounds__(SPLIT_THREADS, HD == 256 ? 2 : 4) q4_keys_kernel(const AttendArgs a) {
  __shared__ Query<HD> query;
  __shared__ int s_max[SPLIT_WARPS];
  griddep_wait();
  griddep_launch();
  Chunk c;
  const bool there = c.find(a);
  if (threadIdx.x < 32) lay_out<HD>(query, a.q + c.b * a.ldq + (long long)c.h * HD);
  if (!there) {
    if (blockIdx.y == 0 && threadIdx.x == 0) nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);  // chunk 0 has slots otherwise
    return;
  }
  const int mx = keys_pass<HD, SPLIT_WARPS>(a, query, c.slot0, c.n, a.logits + c.slot0, [] { __syncthreads(); }, [] {});
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = mx;
  __syncthreads();
  if (threadIdx.x == 0) {
    int m = s_max[0];
    for (int w = 1; w < SPLIT_WARPS; ++w) m = max(m, s_max[w]);
    a.chunk_max[(size_t)c.bh * a.chunks + blockIdx.y] = m;
    if (blockIdx.y == 0) a.arrived[c.bh] = 0;
  }
}

// Each chunk's sum of weights: 4 bytes a slot, from the L2 for the most part.
__global__ void __launch_bounds__(SPLIT_THREADS) q4_sums_kernel(const AttendArgs a) {
  __shared__ int16_t lut[256];
  __shared__ unsigned s_red[SPLIT_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  lut[tid] = d_exp2_lut[tid];
  griddep_wait();
  griddep_launch();
  Chunk c;
  if (!c.find(a)) return;
  int mx = INT_MIN;
  for (int i = lane; i < c.live; i += 32) mx = max(mx, a.chunk_max[(size_t)c.bh * a.chunks + i]);
  mx = __reduce_max_sync(0xffffffffu, mx);
  if (mx == INT_MIN && tid == 0 && blockIdx.y == 0) nsrl_flag(a.st, NSRL_FLAG_ALL_MASKED);
  __syncthreads();
  const unsigned mine = __reduce_add_sync(0xffffffffu, weigh<SPLIT_THREADS>(lut, a.logits + c.slot0, c.n, mx));
  if (lane == 0) s_red[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    unsigned sum = 0;
    for (int w = 0; w < SPLIT_WARPS; ++w) sum += s_red[w];
    a.chunk_sum[(size_t)c.bh * a.chunks + blockIdx.y] = sum;
  }
}

template <int HD>
__global__ void __launch_bounds__(SPLIT_THREADS, HD == 256 ? 2 : 4) q4_values_kernel(const AttendArgs a) {
  using S = Q4Shape<HD>;
  __shared__ __align__(128) uint8_t buffer[SPLIT_WARPS][1024];
  __shared__ int16_t lut[256];
  __shared__ uint32_t recip[128];
  __shared__ long long s_part[SPLIT_WARPS / S::PAIRS][HD];
  __shared__ unsigned s_arrived;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  lut[tid] = d_exp2_lut[tid];
  if (tid < 128) recip[tid] = d_recip_lut[tid];
  griddep_wait();
  griddep_launch();
  Chunk c;
  if (!c.find(a)) return;
  ValuePlaces<HD, true> at(a, c.slot0, a.logits + c.slot0);
  ValueUnit<HD> next;
  first_values<HD, SPLIT_WARPS>(at, c.n, next);
  const unsigned long long flags = flags_of(a);  // the launches before this one have set all there is to set
  // every warp adds up the row's chunks for itself
  int mx = INT_MIN;
  unsigned long long sum = 0;
  for (int i = lane; i < c.live; i += 32) {
    mx = max(mx, a.chunk_max[(size_t)c.bh * a.chunks + i]);
    sum += a.chunk_sum[(size_t)c.bh * a.chunks + i];
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (flags != 0) at.score = nullptr;
  __syncthreads();
  const unsigned inv = mx == INT_MIN ? 0u : reciprocal(recip, sum);
  values_pass<HD, SPLIT_WARPS>(at, next, c.n, lut, mx, inv, buffer[warp], s_part[warp / S::PAIRS]);
  __syncthreads();
  long long total = 0;
  if (tid < HD) {
#pragma unroll
    for (int w = 0; w < SPLIT_WARPS / S::PAIRS; ++w) total += s_part[w][tid];
  }
  if (c.live > 1) {
    // the last chunk to arrive adds up the row's partial contexts
    long long* const row = a.partial + (size_t)c.bh * a.chunks * HD;
    if (tid < HD) row[(size_t)blockIdx.y * HD + tid] = total;
    __threadfence();
    __syncthreads();
    if (tid == 0) s_arrived = atomicAdd(&a.arrived[c.bh], 1u);
    __syncthreads();
    if (s_arrived != (unsigned)c.live - 1) return;
    __threadfence();
    total = 0;
    if (tid < HD)
      for (int r = 0; r < c.live; ++r) total += __ldcg(row + (size_t)r * HD + tid);
  }
  if (tid < HD) a.ctx[c.b * (long long)(a.c.heads * HD) + (long long)c.h * HD + tid] = sat_i16(rhu64(total, 15));
}

template <int HD, int WARPS>
cudaError_t launch_whole(const AttendArgs& a, int parts, size_t share, cudaStream_t s) {
  constexpr int MOST = 4 * (int)(WARPS == 8 ? MANY_SLOTS : MAX_SHARE);
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem((const void*)attend_q4_kernel<HD, WARPS>, MOST, done);
  if (e == cudaSuccess && parts > 8)
    e = cudaFuncSetAttribute(attend_q4_kernel<HD, WARPS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.c.batch * a.c.heads * (size_t)parts));
  cfg.blockDim = dim3(32 * WARPS);
  cfg.dynamicSmemBytes = share * sizeof(int32_t);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, attend_q4_kernel<HD, WARPS>, a);
}

template <int HD>
cudaError_t launch_split(const AttendArgs& a, cudaStream_t s) {
  const dim3 grid((unsigned)(a.c.batch * a.c.heads), (unsigned)a.chunks), block(SPLIT_THREADS);
  cudaError_t e = launch_pdl(q4_keys_kernel<HD>, grid, block, 0, s, a);
  if (e == cudaSuccess) e = launch_pdl(q4_sums_kernel, grid, block, 0, s, a);
  if (e == cudaSuccess) e = launch_pdl(q4_values_kernel<HD>, grid, block, 0, s, a);
  return e;
}

// The form of a call, from what its launch knows (lengths live on the device).
struct Q4Plan {
  bool split, sorted, few;  // few: 8 warps a CTA
  size_t share;             // slots of a CTA of WHOLE, at most
  int parts;                // CTAs of a row
  size_t chunks;            // split: of a row
  size_t logits, chunk_max, chunk_sum, arrived, partial, total;  // scratch offsets and size
};

// WHOLE unless rows are so few that clusters of 16 would be wanted (8 a row
// leave SMs idle) and so long that such a CTA would have over FEW_SLOTS slots:
// clusters of 16 fill the SMs badly.  Microseconds of WHOLE and of split, 64
// dims, scores kept: 8 rows of 131,072 41 and 34, of 65,536 27 and 28; 16 rows
// of 40,960 35 and 30; one row of 262,144 51 and 30; 32 rows of 16,384 22 and 28;
// 64 rows of 16,384 29 and 34; 256 rows of 8,320 39 and 49; 2,048 rows 256 and 330.
//
// A CTA of WHOLE has 8 warps up to FEW_SLOTS slots, and up to MANY_SLOTS where
// rows fill such CTAs one and a half times, 16 otherwise (half as many CTAs an
// SM, half as many steps of a row).  8 and 16: 512 rows of 1,024 x 16 dims 12.8
// and 16.7 us, 512 of 2,048 x 64 25.1 and 27.1; 256 of 8,320 x 64 52 and 39;
// ragged, sorted, 640 of 8,192 56 and 51, 1,024 of 8,192 66 and 72, 2,048 of
// 4,096 70 and 82; equal lengths, 2,048 of 4,096 121 and 130, of 8,320 234 and 231.
//
// From SORT_ROWS rows (two waves of 16 warps) a launch of one CTA sorts the
// sequences by length before.  Sorted and not, ragged: 640 rows of 8,192 51 and 58
// us, 1,280 80 and 97, 2,048 of 8,320 127 and 144; equal lengths: 90.6 and
// 88.5, 234 and 232; 8,192 rows of 128 slots 66.9 and 64.0.  Past SORT_BATCH
// sequences waves are so many that their end counts for little.
//
// Where no head dim is named these are rows of 64 dims, and the limits hold for all:
// at 256 dims an SM has half as many CTAs, so the same numbers of rows are twice as
// many waves there (not measured apart).
//
// Lengths are not seen here: a row takes the form, the CTAs and the shared memory
// of its capacity, however few of its slots are in use.
Q4Plan plan_of(const nsrl_q4_cache& c) {
  Q4Plan p{};
  const size_t bh = c.batch * c.heads;
  p.split = bh * 8 < 148 && c.capacity >= SPLIT_SLOTS;
  p.parts = 1;
  if (!p.split) {
    while (p.parts < MAX_CLUSTER && ((c.capacity + p.parts - 1) / p.parts > MAX_SHARE ||
                                     (bh * p.parts < 148 && c.capacity / p.parts >= 512)))
      p.parts *= 2;
    p.share = ((c.capacity + p.parts - 1) / p.parts + UNIT - 1) / UNIT * UNIT;
    p.few = p.share <= FEW_SLOTS || (bh >= MANY_ROWS && p.share <= MANY_SLOTS);
    p.sorted = bh >= SORT_ROWS && c.batch > 1 && c.batch <= SORT_BATCH;
    if (p.sorted) p.total = c.batch * sizeof(int2);
    return p;
  }
  p.chunks = (c.capacity + CHUNK - 1) / CHUNK;
  auto take = [&](size_t n) {
    const size_t at = p.total;
    p.total += (n + 255) & ~size_t(255);
    return at;
  };
  p.logits = take(bh * c.capacity * sizeof(int32_t));
  p.chunk_max = take(bh * p.chunks * sizeof(int32_t));
  p.chunk_sum = take(bh * p.chunks * sizeof(unsigned));
  p.arrived = take(bh * sizeof(unsigned));
  p.partial = take(bh * p.chunks * c.head_dim * sizeof(long long));
  return p;
}

}  // namespace

size_t q4_max_capacity() { return 8 * MAX_SHARE; }

size_t q4_attend_workspace(const nsrl_q4_cache& c) { return plan_of(c).total; }

cudaError_t launch_attend_q4(const int16_t* q, size_t ldq, const nsrl_q4_cache& c, const int32_t* lens, int len_offset,
                             int16_t* ctx, void* ws, nsrl_device_status* st, cudaStream_t s) {
  const size_t bh = c.batch * c.heads;
  if (bh == 0) return cudaSuccess;
  if (c.capacity > q4_max_capacity() || bh > 0x7fffffffull / MAX_CLUSTER) return cudaErrorInvalidValue;
  AttendArgs a{};
  a.c = c;
  a.q = q;
  a.ldq = (long long)ldq;
  a.lens = lens;
  a.len_offset = len_offset;
  a.ctx = ctx;
  a.st = st;
  const Q4Plan p = plan_of(c);
  const double slots = (double)bh * (double)c.capacity;
  ProfScope prof("attention_decode_q4", s, 4.0 * slots * (double)c.head_dim,
                 slots * ((double)c.head_dim + 8.0 * std::max<size_t>(1, c.head_dim / 32) + (c.scores ? 8.0 : 0.0)));
  cudaError_t e;
  if (p.split) {
    uint8_t* base = static_cast<uint8_t*>(ws);
    a.chunks = (int)p.chunks;
    a.logits = reinterpret_cast<int32_t*>(base + p.logits);
    a.chunk_max = reinterpret_cast<int32_t*>(base + p.chunk_max);
    a.chunk_sum = reinterpret_cast<unsigned*>(base + p.chunk_sum);
    a.arrived = reinterpret_cast<unsigned*>(base + p.arrived);
    a.partial = reinterpret_cast<long long*>(base + p.partial);
    e = c.head_dim == 16 ? launch_split<16>(a, s) : c.head_dim == 64 ? launch_split<64>(a, s) : launch_split<256>(a, s);
  } else {
    const size_t share = p.share;
    const bool few = p.few;
    if (p.sorted) {
      a.order = static_cast<int2*>(ws);
      while (c.capacity >> a.length_shift >= LENGTHS) ++a.length_shift;
      e = launch_pdl(q4_order_kernel, dim3(1), dim3(1024), 0, s, a);
      if (e != cudaSuccess) return e;
    } else if (c.scores && c.batch > SORT_BATCH) {
      e = launch_pdl(q4_screen_kernel, dim3((unsigned)((c.batch + 255) / 256)), dim3(256), 0, s, a);
      if (e != cudaSuccess) return e;
    }
    a.lens_known = p.sorted || c.batch > SORT_BATCH;
    e = c.head_dim == 16   ? (few ? launch_whole<16, 8>(a, p.parts, share, s) : launch_whole<16, 16>(a, p.parts, share, s))
        : c.head_dim == 64 ? (few ? launch_whole<64, 8>(a, p.parts, share, s) : launch_whole<64, 16>(a, p.parts, share, s))
                           : (few ? launch_whole<256, 8>(a, p.parts, share, s) : launch_whole<256, 16>(a, p.parts, share, s));
  }
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace nsrl
