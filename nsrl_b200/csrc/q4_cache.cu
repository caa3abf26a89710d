// The 4-bit KV cache: append (quantise), read (dequantise) and eviction by
// accumulated attention weight.  The format is described in nsrl_b200.h.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace nsrl {
namespace {

constexpr int THREADS = 256;

// ---------------------------------------------------------- append, read ---
// Append: a thread owns 16 dims of one (sequence, head, token), of the key and of
// the value: a 32-byte sector of int16 and 8 bytes of codes each.  Threads run
// over dims, then tokens, then heads, so a warp's cache rows are contiguous.
// Memory has 4 hd bytes of int16 and hd + 8 ceil(hd / 32) of cache to move per
// slot; append is bound by its instructions, half of them for the row and its
// scales: 8 prompts of up to 2,048 tokens, 8 x 64 dims, take 10.8 us, and 13.4
// with 8 dims a thread.
struct AppendArgs {
  nsrl_q4_cache c;
  const int16_t* k;
  const int16_t* v;
  long long ld;
  long long tokens;
  unsigned rows;  // batch * heads * tokens
  const int32_t* starts;
  const int32_t* counts;
  const int32_t* positions;
  nsrl_device_status* st;
};

__device__ __forceinline__ uint4 load8(const int16_t* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)(uint16_t)p[2 * i] | ((uint32_t)(uint16_t)p[2 * i + 1] << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Sixteen dims to sixteen codes; scale_word is the group's (two lanes of the
// warp, one where PAIRED is false).
template <bool PAIRED>
__device__ __forceinline__ uint2 quantise16(const uint4 (&u)[2], uint32_t& scale_word) {
  // smallest values and smallest complements (so the largest values), two at a time
  auto least = [](const uint4& v) { return __vmins2(__vmins2(v.x, v.y), __vmins2(v.z, v.w)); };
  auto most = [](const uint4& v) { return __vmaxs2(__vmaxs2(v.x, v.y), __vmaxs2(v.z, v.w)); };
  const uint32_t low = __vmins2(least(u[0]), least(u[1])), high = __vmaxs2(most(u[0]), most(u[1]));
  uint32_t both = __vmins2(__byte_perm(low, ~high, 0x5410), __byte_perm(low, ~high, 0x7632));
  if (PAIRED) both = __vmins2(both, __shfl_xor_sync(0xffffffffu, both, 1));
  const int lo = (int)(int16_t)(both & 0xFFFF), hi = ~((int)both >> 16);
  const unsigned scale = max(1u, (unsigned)(hi - lo + 14) / 15u);
  // floor(n / d) = n * ceil(2^32 / d) >> 32 while n d < 2^32 (Granlund and
  // Montgomery): n = 2 (x - lo) + scale < 2^17.1, d = 2 scale < 2^13.1
  const unsigned d = 2 * scale;
  const unsigned magic = 0xFFFFFFFFu / d + 1;
  const int offset = (int)scale - 2 * lo;
  const bool top = hi + (int)(scale / 2) > 32767;  // a value may pass 32767: its code goes one down
  uint32_t codes[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    int x[8];
    unpack8(u[e], x);
    uint32_t w = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) w = w * 16 + __umulhi((unsigned)(2 * x[i] + offset), magic);
    if (top)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (lo + (int)(scale * ((w >> (4 * i)) & 15)) > 32767) w -= 1u << (4 * i);
    codes[e] = w;
  }
  scale_word = scale | ((uint32_t)lo << 16);
  return make_uint2(codes[0], codes[1]);
}

template <int HD>
__global__ void __launch_bounds__(THREADS) q4_append_kernel(const AppendArgs a, const bool vec) {
  constexpr int LPR = HD / 16;               // lanes of a row
  constexpr int LPG = HD < 32 ? 1 : 2;       // lanes of a group
  constexpr int G = HD < 32 ? 1 : HD / 32;
  griddep_wait();
  griddep_launch();
  const int sub = threadIdx.x % LPR;
  const unsigned row = blockIdx.x * (THREADS / LPR) + threadIdx.x / LPR;
  const bool inside = row < a.rows;  // every lane of a warp takes part in the shuffles
  const unsigned tokens = (unsigned)a.tokens, heads = (unsigned)a.c.heads;
  const unsigned bh = inside ? row / tokens : 0, t = inside ? row - bh * tokens : 0;
  const unsigned b = bh / heads, h = bh - b * heads;
  const long long start = a.starts[b], count = a.counts ? (long long)a.counts[b] : a.tokens;
  const bool fits = start >= 0 && count >= 0 && count <= a.tokens && start + count <= (long long)a.c.capacity;
  if (inside && !fits && t == 0 && sub == 0 && h == 0) nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
  const bool live = inside && fits && (long long)t < count;
  if (!__any_sync(0xffffffffu, live)) return;
  uint4 uk[2] = {}, uv[2] = {};
  if (live) {
    const long long off = ((long long)b * a.tokens + t) * a.ld + (long long)h * HD + 16 * sub;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uk[e] = load8(a.k + off + 8 * e, vec);
      uv[e] = load8(a.v + off + 8 * e, vec);
    }
  }
  uint32_t sk, sv;
  const uint2 ck = quantise16<LPG == 2>(uk, sk), cv = quantise16<LPG == 2>(uv, sv);
  if (!live) return;
  const size_t slot = (size_t)bh * a.c.capacity + (size_t)(start + t);
  reinterpret_cast<uint2*>(a.c.k_codes)[slot * LPR + sub] = ck;
  reinterpret_cast<uint2*>(a.c.v_codes)[slot * LPR + sub] = cv;
  if (sub % LPG == 0) {
    a.c.k_scales[slot * G + sub / LPG] = sk;
    a.c.v_scales[slot * G + sub / LPG] = sv;
  }
  if (sub == 0) {
    if (a.c.scores) a.c.scores[slot] = 0;
    if (a.c.positions) a.c.positions[slot] = (int32_t)((a.positions ? (long long)a.positions[b] : start) + t);
  }
}

struct ReadArgs {
  nsrl_q4_cache c;
  const int32_t* starts;
  long long tokens;
  unsigned rows;
  int16_t* k;
  int16_t* v;
  nsrl_device_status* st;
};

__device__ __forceinline__ uint4 dequantise8(uint32_t codes, uint32_t scale_word) {
  const int scale = (int)(scale_word & 0xFFFF), zero = (int)(int16_t)(scale_word >> 16);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = pack_sat16(zero + scale * (int)((codes >> (8 * i + 4)) & 15), zero + scale * (int)((codes >> (8 * i)) & 15));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Read: a lane takes pieces of 8 dims, half a row apart where a row has more than
// two, so that four accesses are under way and each store of a warp fills whole
// sectors.  2,048 rows of 2,048 slots take 211 us, all of the copy bandwidth (218
// with two rows of 8 dims a thread, 245 with one).
template <int HD>
struct ReadShape {
  static constexpr int E = HD == 16 ? 1 : 2;          // pieces of a lane
  static constexpr int LPR = HD / (8 * E);            // lanes of a row
  static constexpr int ROWS = THREADS / LPR;          // rows of a block
};

template <int HD>
__global__ void __launch_bounds__(THREADS) q4_read_kernel(const ReadArgs a) {
  using S = ReadShape<HD>;
  constexpr int G = HD < 32 ? 1 : HD / 32, PPG = HD < 32 ? HD / 8 : 4;  // groups, pieces of a group
  constexpr int E = S::E, LPR = S::LPR;
  griddep_wait();
  griddep_launch();
  const int sub = threadIdx.x % LPR;
  const unsigned row = blockIdx.x * S::ROWS + threadIdx.x / LPR;
  if (row >= a.rows) return;
  const unsigned tokens = (unsigned)a.tokens;
  const unsigned bh = row / tokens, t = row - bh * tokens, b = bh / (unsigned)a.c.heads;
  const long long start = a.starts ? (long long)a.starts[b] : 0;
  if (start < 0 || start + a.tokens > (long long)a.c.capacity) {
    if (t == 0 && sub == 0) nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
    return;
  }
  const size_t slot = (size_t)bh * a.c.capacity + (size_t)(start + t);
  uint32_t ck[E], cv[E], sk[E], sv[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int piece = sub + LPR * e;
    ck[e] = reinterpret_cast<const uint32_t*>(a.c.k_codes)[slot * (HD / 8) + piece];
    cv[e] = reinterpret_cast<const uint32_t*>(a.c.v_codes)[slot * (HD / 8) + piece];
    sk[e] = a.c.k_scales[slot * G + piece / PPG];
    sv[e] = a.c.v_scales[slot * G + piece / PPG];
  }
  const size_t i = (size_t)row * (HD / 8) + sub;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    reinterpret_cast<uint4*>(a.k)[i + LPR * e] = dequantise8(ck[e], sk[e]);
    reinterpret_cast<uint4*>(a.v)[i + LPR * e] = dequantise8(cv[e], sv[e]);
  }
}

// ------------------------------------------------------------- eviction ----
// Two launches.  q4_select_kernel (one CTA per (sequence, head)) finds the
// keep-th largest key by radix selection, 8 bits a pass from the highest bit in
// use and no further than the bin that is kept whole, where key = 2^31 for a
// protected slot, else max(score, 0); marks the kept slots (ties to the lower
// slot) in a shared-memory bitmap; lists the holes below `keep` and the kept
// slots at or past it, both in ascending order and equally many.
// q4_move_kernel copies the m-th listed slot into the m-th hole.  Sources lie
// at or past `keep` and destinations below it, so the moves need no order.
constexpr unsigned SAFE = 0x80000000u;  // key of a protected slot, above every score
constexpr int SELECT_HELD = 16;         // keys of a lane in registers
constexpr int SELECT_WARPS = 20;        // of a CTA, at most: 48 registers a thread

struct EvictArgs {
  nsrl_q4_cache c;
  const int32_t* lens;
  const int32_t* next;
  long long keep, sinks, recent, most;  // most: moves a (sequence, head) can have
  int32_t* scores_out;
  int32_t* positions_out;
  int32_t* lens_out;
  int32_t* moves;  // [batch * heads]
  int2* list;      // [batch * heads][most]: (from, to)
  nsrl_device_status* st;
};

// The first HELD keys of a lane stay in registers (loaded all at once: the loads'
// latency is most of a short row's time); a longer span's others are made again in
// each pass, and scores and positions are read again where they are copied.
// Bound by instructions (some 126 a round of 32 slots at three passes, ties among
// the last) and the barriers between passes, well above its 8 bytes a slot in and
// 8 a kept slot out: 2,048 rows of 2,112 slots take 40 us, their bytes 10.
__global__ void __launch_bounds__(32 * SELECT_WARPS, 2) q4_select_kernel(const EvictArgs a) {
  constexpr int HELD = SELECT_HELD, STEP = 4;  // keys are gone through STEP rounds at a time
  extern __shared__ uint32_t bitmap[];         // kept slots, 32 a word
  __shared__ int hist[256 + 32];  // and a place a lane for keys that are not counted
  __shared__ int warp_a[SELECT_WARPS], warp_b[SELECT_WARPS];
  __shared__ unsigned s_prefix, s_top;
  __shared__ int s_want, s_safe;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int threads = blockDim.x, warps = threads >> 5;
  if (tid == 0) {
    s_top = 0;
    s_safe = 0;
  }
  for (int i = tid; i < 256; i += threads) hist[i] = 0;
  griddep_wait();
  griddep_launch();
  const unsigned bh = blockIdx.x, b = bh / (unsigned)a.c.heads;
  const int keep = (int)a.keep;
  const int n = a.lens[b];
  if (n < 0 || n > (int)a.c.capacity) {
    if (tid == 0) {
      nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
      a.moves[bh] = 0;
    }
    return;
  }
  const size_t base = (size_t)bh * a.c.capacity;
  const int32_t* scores = a.c.scores + base;
  const int32_t* positions = a.c.positions + base;
  int32_t* scores_out = a.scores_out + base;
  int32_t* positions_out = a.positions_out + base;
  if (n <= keep) {
    for (int i = tid; i < n; i += threads) {
      scores_out[i] = scores[i];
      positions_out[i] = positions[i];
    }
    if (tid == 0) a.moves[bh] = 0;
    return;
  }
  // protected: positions up to sink, and from border on
  const int sink = (int)min(a.sinks - 1, (long long)INT_MAX);
  const int border = (int)max((long long)a.next[b] - a.recent, (long long)INT_MIN);
  // Each warp takes one contiguous span of slots, 32 at a time, so that ranks
  // follow the slot order.
  const int span = ((n + warps - 1) / warps + 31) / 32 * 32;
  const int lo = min(n, warp * span), hi = min(n, lo + span);
  const int rounds = (hi - lo + 31) / 32;
  auto key_of = [&](int score, int position) -> unsigned {
    return position <= sink || position >= border ? SAFE : (unsigned)max(score, 0);
  };
  const int32_t* my_scores = scores + lo + lane;
  const int32_t* my_positions = positions + lo + lane;
  const int mine = hi - lo - lane;  // this lane's slot of round r is there if 32 r < mine
  // A round past the span, or a slot past the row's end, has the smallest key, 0:
  // counts of larger keys do not see it.  Where equal keys count, `mine` leaves it out.
  unsigned key[HELD];
  {
    int score[HELD], position[HELD];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      score[k] = 32 * k < mine ? my_scores[32 * k] : 0;
      position[k] = 32 * k < mine ? my_positions[32 * k] : 0;
    }
#pragma unroll
    for (int k = 0; k < HELD; ++k) key[k] = 32 * k < mine ? key_of(score[k], position[k]) : 0;
  }
  // f(round, key) for every round of the warp's span, and for some past it
  auto each = [&](auto f) {
#pragma unroll
    for (int k = 0; k < HELD; k += STEP)
      if (k < rounds) {
#pragma unroll
        for (int m = 0; m < STEP; ++m) f(k + m, key[k + m]);
      }
    for (int k = HELD; k < rounds; ++k) f(k, 32 * k < mine ? key_of(my_scores[32 * k], my_positions[32 * k]) : 0);
  };

  // ---- the protected slots, and the largest other key ----
  int safe = 0;
  unsigned top = 0;
  each([&](int, unsigned k) {
    safe += (int)(k >> 31);
    top = max(top, k & ~SAFE);
  });
  safe = __reduce_add_sync(0xffffffffu, safe);
  top = __reduce_max_sync(0xffffffffu, top);
  __syncthreads();
  if (lane == 0) {
    atomicAdd(&s_safe, safe);
    atomicMax(&s_top, top);
  }
  __syncthreads();
  // ---- the last key that stays: kept are the keys above it, and the first `want` slots that equal it ----
  unsigned last = SAFE;
  int want = keep;
  if (s_safe < keep) {
    want = keep - s_safe;
    unsigned prefix = 0;
    int shift = s_top == 0 ? 0 : max(0, 24 - __clz(s_top));  // the top eight bits in use first
    int fixed = 31;  // the bits of `prefix` from here up are settled (SAFE has bit 31, `prefix` has not)
    for (;;) {
      each([&](int, unsigned k) {
        atomicAdd(&hist[(k ^ prefix) >> fixed ? 256 + lane : (k >> shift) & 255], 1);
      });
      __syncthreads();
      if (warp == 0) {
        // lane l holds bins 255 - 8 l down to 248 - 8 l: a scan from the top
        int own[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          own[j] = hist[255 - 8 * lane - j];
          sum += own[j];
        }
        int before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += v;
        }
        before -= sum;  // keys in higher bins of other lanes
        if (before < want && before + sum >= want) {  // one lane: its bins hold the want-th key
          int j = 0;
          while (before + own[0] < want) {
            before += own[0];
#pragma unroll
            for (int m = 0; m < 7; ++m) own[m] = own[m + 1];
            ++j;
          }
          s_prefix = (prefix & ~(255u << shift)) | (unsigned)(255 - 8 * lane - j) << shift;
          s_want = want - before;
          s_top = (unsigned)own[0];
        }
      }
      __syncthreads();
      prefix = s_prefix;
      want = s_want;
      const bool all = want == (int)s_top;  // every key of the bin stays: what lies above prefix - 1
      if (all && prefix > 0) {
        last = prefix - 1;
        want = 0;
        break;
      }
      if (shift == 0) {
        last = prefix;
        break;
      }
      fixed = shift;
      shift = max(0, shift - 8);
      for (int i = tid; i < 256; i += threads) hist[i] = 0;
      __syncthreads();
    }
  }

  auto prefix_of_warps = [&](int mine) {  // exclusive prefix over the warps of lane w's count of warp w
    int before = lane < warp ? mine : 0;
    return __reduce_add_sync(0xffffffffu, before);
  };
  const unsigned under = (1u << lane) - 1;
  int cutoff = lo;   // of the slots whose key is `last`, those below it stay: ties go to the lower slots
  if (want > 0) {
    int equal = 0;
    each([&](int r, unsigned k) { equal += k == last && 32 * r < mine; });
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) warp_a[warp] = equal;
    __syncthreads();
    int rank = prefix_of_warps(lane < warps ? warp_a[lane] : 0);
    __syncthreads();
    if (rank + equal <= want)
      cutoff = hi;
    else if (rank < want) {  // this warp has the last of them
      each([&](int r, unsigned k) {
        const bool tie = k == last && 32 * r < mine;
        const unsigned eq = __ballot_sync(0xffffffffu, tie);
        if (tie && rank + __popc(eq & under) < want) cutoff = lo + 32 * r + lane + 1;
        rank += __popc(eq);
      });
      cutoff = __reduce_max_sync(0xffffffffu, cutoff);
    }
  }
  const bool copy_scores = scores_out != scores, copy_positions = positions_out != positions;
  int32_t* my_scores_out = scores_out + lo + lane;
  int32_t* my_positions_out = positions_out + lo + lane;
  const int ties = cutoff - lo - lane, low = min(keep, hi) - lo - lane;
  each([&](int r, unsigned k) {
    const bool kept = k > last || (k == last && 32 * r < ties);
    const unsigned bits = __ballot_sync(0xffffffffu, kept);
    if (lane == 0 && r < rounds) bitmap[(lo >> 5) + r] = bits;
    if (kept && 32 * r < low) {
      if (copy_scores) my_scores_out[32 * r] = my_scores[32 * r];
      if (copy_positions) my_positions_out[32 * r] = my_positions[32 * r];
    }
  });
  __syncwarp();
  // A lane takes a word of the warp's part of the bitmap: its holes below `keep`, and its kept slots at or past it.
  auto word = [&](int r, unsigned& hole, unsigned& late) {
    const int first = lo + 32 * r;
    const unsigned bits = r < rounds ? bitmap[first >> 5] : 0;
    const int low = max(0, min(32, keep - first)), live = max(0, min(32, hi - first));
    const unsigned low_mask = low >= 32 ? 0xffffffffu : (1u << low) - 1;
    const unsigned live_mask = live >= 32 ? 0xffffffffu : (1u << live) - 1;
    hole = ~bits & low_mask & live_mask;
    late = bits & ~low_mask;
  };
  int holes = 0, lates = 0;
  for (int r = lane; r < rounds; r += 32) {
    unsigned hole, late;
    word(r, hole, late);
    holes += __popc(hole);
    lates += __popc(late);
  }
  holes = __reduce_add_sync(0xffffffffu, holes);
  lates = __reduce_add_sync(0xffffffffu, lates);
  if (lane == 0) {
    warp_a[warp] = holes;
    warp_b[warp] = lates;
  }
  __syncthreads();
  int hole_rank = prefix_of_warps(lane < warps ? warp_a[lane] : 0);
  int late_rank = prefix_of_warps(lane < warps ? warp_b[lane] : 0);
  int2* list = a.list + (size_t)bh * a.most;
  for (int r0 = 0; r0 < rounds; r0 += 32) {
    unsigned hole, late;
    word(r0 + lane, hole, late);
    // both counts in one scan: at most 1,024 each
    const unsigned both = (unsigned)__popc(hole) | (unsigned)__popc(late) << 16;
    unsigned upto = both;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned total = __shfl_sync(0xffffffffu, upto, 31);
    const int first = lo + 32 * (r0 + lane);
    int at = hole_rank + (int)((upto - both) & 0xFFFF);
    for (; hole; hole &= hole - 1) list[at++].y = first + __ffs((int)hole) - 1;
    at = late_rank + (int)((upto - both) >> 16);
    for (; late; late &= late - 1) list[at++].x = first + __ffs((int)late) - 1;
    hole_rank += (int)(total & 0xFFFF);
    late_rank += (int)(total >> 16);
  }
  if (tid == threads - 1) a.moves[bh] = late_rank;  // the last warp's running rank is the total
}

// A move is 2 head_dim / 2 code bytes, the scales, the score and the position:
// 88 bytes at 64 dims, in pieces of 16, 8 and 4 bytes, one a lane, LANES lanes
// a move, and UNROLL moves of a lane in flight.  Few bytes, three dependent
// accesses (list, source, store): 15 us for 64 moves of each of 2,048 rows.
template <int HD>
__global__ void __launch_bounds__(THREADS) q4_move_kernel(const EvictArgs a) {
  constexpr int LANES = HD == 256 ? 32 : 8, UNROLL = 4, PER = THREADS / LANES;
  constexpr int CODE = HD / 2;                         // bytes of a slot's codes in one tensor
  constexpr int SCALE = HD < 32 ? 4 : HD / 8;          // and of its scales
  constexpr int CB = CODE < 16 ? CODE : 16, SB = SCALE < 16 ? SCALE : 16;  // piece sizes
  constexpr int CN = CODE / CB, SN = SCALE / SB;       // pieces
  static_assert(2 * CN + 2 * SN + 2 <= LANES);
  griddep_wait();
  griddep_launch();
  const unsigned bh = blockIdx.x;
  const int moves = a.moves[bh];
  const size_t base = (size_t)bh * a.c.capacity;
  // this lane's piece: where it comes from, where it goes, bytes, stride of a slot
  const int piece = threadIdx.x % LANES;
  const uint8_t* src = nullptr;
  uint8_t* dst = nullptr;
  int bytes = 0, stride = 0;
  auto take = [&](const void* from, void* to, int size, int slot_bytes, int offset) {
    src = static_cast<const uint8_t*>(from) + base * slot_bytes + offset;
    dst = static_cast<uint8_t*>(to) + base * slot_bytes + offset;
    bytes = size;
    stride = slot_bytes;
  };
  if (piece < CN)
    take(a.c.k_codes, a.c.k_codes, CB, CODE, CB * piece);
  else if (piece < 2 * CN)
    take(a.c.v_codes, a.c.v_codes, CB, CODE, CB * (piece - CN));
  else if (piece < 2 * CN + SN)
    take(a.c.k_scales, a.c.k_scales, SB, SCALE, SB * (piece - 2 * CN));
  else if (piece < 2 * CN + 2 * SN)
    take(a.c.v_scales, a.c.v_scales, SB, SCALE, SB * (piece - 2 * CN - SN));
  else if (piece == 2 * CN + 2 * SN)
    take(a.c.scores, a.scores_out, 4, 4, 0);
  else if (piece == 2 * CN + 2 * SN + 1)
    take(a.c.positions, a.positions_out, 4, 4, 0);
  const int2* list = a.list + (size_t)bh * a.most;
  for (int m0 = blockIdx.y * PER * UNROLL; m0 < moves; m0 += gridDim.y * PER * UNROLL) {
    int2 e[UNROLL];
    uint4 v[UNROLL];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int m = m0 + k * PER + threadIdx.x / LANES;
      e[k] = m < moves && bytes ? list[m] : make_int2(-1, -1);
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      if (e[k].x < 0) continue;
      const uint8_t* s = src + (size_t)e[k].x * stride;
      if (bytes == 16)
        v[k] = *reinterpret_cast<const uint4*>(s);
      else if (bytes == 8)
        *reinterpret_cast<uint2*>(&v[k]) = *reinterpret_cast<const uint2*>(s);
      else
        v[k].x = *reinterpret_cast<const uint32_t*>(s);
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      if (e[k].x < 0) continue;
      uint8_t* d = dst + (size_t)e[k].y * stride;
      if (bytes == 16)
        *reinterpret_cast<uint4*>(d) = v[k];
      else if (bytes == 8)
        *reinterpret_cast<uint2*>(d) = make_uint2(v[k].x, v[k].y);
      else
        *reinterpret_cast<uint32_t*>(d) = v[k].x;
    }
  }
  // lens_out may be lens, so it changes only after the selection has read it
  if (blockIdx.y == 0 && bh % (unsigned)a.c.heads == 0 && threadIdx.x == 0) {
    const unsigned b = bh / (unsigned)a.c.heads;
    const int n = a.lens[b];
    if (n >= 0 && n <= (int)a.c.capacity) a.lens_out[b] = min(n, (int)a.keep);
  }
}

size_t most_moves(const nsrl_q4_cache& c, size_t keep) { return std::min(keep, c.capacity - keep); }
size_t list_offset(const nsrl_q4_cache& c) { return (c.batch * c.heads * sizeof(int32_t) + 255) & ~size_t(255); }

}  // namespace

cudaError_t launch_q4_append(const nsrl_q4_cache& c, const int16_t* k, const int16_t* v, size_t ld, size_t tokens,
                             const int32_t* starts, const int32_t* counts, const int32_t* positions,
                             nsrl_device_status* st, cudaStream_t s) {
  const size_t n = c.batch * c.heads * tokens, per_block = THREADS / (c.head_dim / 16);
  if (n == 0) return cudaSuccess;
  if (n > 0xffffff00u) return cudaErrorInvalidValue;  // the entry point refuses it
  const AppendArgs a{c, k, v, (long long)ld, (long long)tokens, (unsigned)n, starts, counts, positions, st};
  const bool vec = ld % 8 == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  const double rows = (double)(c.batch * c.heads) * (double)tokens;
  ProfScope prof("q4_append", s, 0.0, rows * (4.0 * c.head_dim + c.head_dim + 8.0 * std::max<size_t>(1, c.head_dim / 32)));
  auto* kernel = c.head_dim == 16 ? q4_append_kernel<16> : c.head_dim == 64 ? q4_append_kernel<64> : q4_append_kernel<256>;
  const cudaError_t e = launch_pdl(kernel, dim3((unsigned)((n + per_block - 1) / per_block)), dim3(THREADS), 0, s, a, vec);
  return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_q4_read(const nsrl_q4_cache& c, const int32_t* starts, size_t tokens, int16_t* k, int16_t* v,
                           nsrl_device_status* st, cudaStream_t s) {
  const size_t n = c.batch * c.heads * tokens;
  const size_t per_block = c.head_dim == 16   ? ReadShape<16>::ROWS
                           : c.head_dim == 64 ? ReadShape<64>::ROWS
                                              : ReadShape<256>::ROWS;
  if (n == 0) return cudaSuccess;
  if (n > 0xffffff00u) return cudaErrorInvalidValue;  // the entry point refuses it
  const ReadArgs a{c, starts, (long long)tokens, (unsigned)n, k, v, st};
  const double rows = (double)(c.batch * c.heads) * (double)tokens;
  ProfScope prof("q4_read", s, 0.0, rows * (4.0 * c.head_dim + c.head_dim + 8.0 * std::max<size_t>(1, c.head_dim / 32)));
  auto* kernel = c.head_dim == 16 ? q4_read_kernel<16> : c.head_dim == 64 ? q4_read_kernel<64> : q4_read_kernel<256>;
  const cudaError_t e = launch_pdl(kernel, dim3((unsigned)((n + per_block - 1) / per_block)), dim3(THREADS), 0, s, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

size_t q4_evict_workspace(const nsrl_q4_cache& c, size_t keep) {
  return list_offset(c) + c.batch * c.heads * most_moves(c, keep) * sizeof(int2);
}

cudaError_t launch_q4_evict(const nsrl_q4_cache& c, const int32_t* lens, const int32_t* next, size_t keep, size_t sinks,
                            size_t recent, int32_t* scores_out, int32_t* positions_out, int32_t* lens_out, void* ws,
                            nsrl_device_status* st, cudaStream_t s) {
  const size_t bh = c.batch * c.heads;
  if (bh == 0) return cudaSuccess;
  EvictArgs a{};
  a.c = c;
  a.lens = lens;
  a.next = next;
  a.keep = (long long)keep;
  a.sinks = (long long)sinks;
  a.recent = (long long)recent;
  a.most = (long long)most_moves(c, keep);
  a.scores_out = scores_out;
  a.positions_out = positions_out;
  a.lens_out = lens_out;
  a.moves = static_cast<int32_t*>(ws);
  a.list = reinterpret_cast<int2*>(static_cast<uint8_t*>(ws) + list_offset(c));
  a.st = st;
  const size_t smem = (c.capacity / 32 + 1) * sizeof(uint32_t);
  {
    // Warps follow the capacity, one for the keys that its lanes hold, four at least.
    const size_t warps = std::min<size_t>(SELECT_WARPS, std::max<size_t>(4, (c.capacity + 32 * SELECT_HELD - 1) / (32 * SELECT_HELD)));
    ProfScope prof("q4_select", s, 0.0, 8.0 * (double)bh * (double)c.capacity);
    // the bitmap of the largest capacity is 32 KB: within the default limit
    const cudaError_t e = launch_pdl(q4_select_kernel, dim3((unsigned)bh), dim3(32 * (unsigned)warps), smem, s, a);
    if (e != cudaSuccess) return e;
  }
  // moves of a CTA's step: 128 (32 at 256 dims), as many CTAs a row as its moves may need, 64 at most
  const size_t step = c.head_dim == 256 ? 32 : 128;
  const unsigned chunks = (unsigned)std::max<size_t>(1, std::min<size_t>((a.most + step - 1) / step, 64));
  ProfScope prof("q4_move", s, 0.0, 2.0 * (double)bh * (double)a.most * (double)c.head_dim);
  auto* kernel = c.head_dim == 16 ? q4_move_kernel<16> : c.head_dim == 64 ? q4_move_kernel<64> : q4_move_kernel<256>;
  const cudaError_t e = launch_pdl(kernel, dim3((unsigned)bh, chunks), dim3(THREADS), 0, s, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace nsrl
