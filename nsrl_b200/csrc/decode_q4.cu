// Attention of one query per sequence over the 4-bit cache
// (nsrl_attention_decode_q4): the logits, base-2 softmax and context of
// nsrl_attention_decode (attention.cu) on the values the codes stand for.
//
// With value = zero + scale * code per group g of 32 dims,
//   q . k   = sum_g scale_g (sum_i q_i code_i) + zero_g (sum_i q_i)
//   sum p v = sum_j p_j zero_jg + (p_j scale_jg) code_j.
//
// The Q15 weights need the row's maximum and sum before the first value is
// weighed, so a (sequence, head) is one cluster of CTAs: each takes a
// contiguous share of the slots, keeps their logits in shared memory, and the
// cluster exchanges maximum, sum and partial contexts through distributed
// shared memory (maximum and sum by a store and an arrival on every CTA's own
// barrier, so that the copying warp takes no part).  The cache is read once.
//
// Bound by memory (80 bytes a slot of 64 dims, 88 with scores) as long as an
// SM spends below about 3.5 cycles on a slot, which IMADs on unpacked codes do
// not (128 of them a slot).  So both products are int8 MMAs (m16n8k32) on codes
// widened to bytes, exact in s32:
//   keys:   A = 16 slots x 32 dims of one group; B = the query's planes of that
//           group, q = 256 h + l + 128 with h, l in s8, and ones for the sum of
//           the codes.  Groups 2i and 2i + 1 use columns 0..2 and 4..6 of one
//           accumulator, so a quad's lanes hold the two groups' parts.
//   values: A = 16 dims x 32 slots (a 4 x 4 byte transpose by PRMT); B = the
//           four byte planes of p_j scale_jg of two groups, one column each.
// Warp 8 streams tiles of codes and scales (K, then V) through a ring of bulk
// copies, so value tiles arrive while the softmax runs; warps 0..7 consume them.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstdlib>

#include "common.cuh"
#include "internal.h"

namespace cg = cooperative_groups;

namespace nsrl {
namespace {

constexpr int WARPS = 8, CONSUMERS = 32 * WARPS, THREADS = CONSUMERS + 32;
constexpr int MAX_CLUSTER = 8;
constexpr int SHARE_UNIT = 32;       // slots of a value MMA
constexpr size_t MAX_SHARE = 32768;  // logits of a CTA: 128 KB

template <int HD>
struct Q4Shape {
  static constexpr int WORDS = HD / 8;                   // code words of a slot
  static constexpr int G = HD < 32 ? 1 : HD / 32;        // groups
  static constexpr int PAIRS = (G + 1) / 2;              // pairs of groups, 64 dims each
  static constexpr int SHIFT = HD == 16 ? 2 : HD == 64 ? 3 : 4;
  static constexpr int TILE = HD == 16 ? 512 : HD == 64 ? 256 : 128;  // slots of a stage
  static constexpr int UNIT = HD == 256 ? 16 : 32;  // slots of a warp's step through the keys
  static constexpr int STAGES = HD == 256 ? 3 : 4;
  static constexpr int CODE_BYTES = TILE * HD / 2, SCALE_BYTES = TILE * G * 4;
  static constexpr int STAGE_BYTES = CODE_BYTES + SCALE_BYTES;
};

struct AttendArgs {
  nsrl_q4_cache c;
  const int16_t* q;
  long long ldq;
  const int32_t* lens;
  int len_offset;
  int16_t* ctx;
  nsrl_device_status* st;
};

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(CONSUMERS) : "memory"); }

// Untiled bulk copy global -> shared, both 16-byte aligned, a multiple of 16 bytes.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Gives `value` to slot `part` of every CTA of the cluster and waits (bounded)
// until all `parts` values are here.  All consumer threads call it with the
// same `values` and `bar`; lane r of warp 0 serves rank r.
template <typename T>
__device__ __forceinline__ bool exchange(const cg::cluster_group& cluster, T* values, uint64_t* bar, T value, int part,
                                         int parts, nsrl_device_status* st) {
  if ((int)threadIdx.x < parts) {
    cluster.map_shared_rank(values, threadIdx.x)[part] = value;
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(bar)), "r"(threadIdx.x));
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
  }
  const unsigned long long t0 = global_ns();
  for (uint32_t i = 0;; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0, %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(20000u)
        : "memory");
    if (ok) return true;
    if ((i & 15u) == 15u && global_ns() - t0 > NSRL_WAIT_NS) {
      nsrl_flag(st, NSRL_FLAG_WAIT_TIMEOUT);
      return false;
    }
  }
}

__device__ __forceinline__ void mma_u8s8(int (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
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

constexpr uint32_t LOW = 0x0F0F0F0Fu, HIGH = 0xF0F0F0F0u;

// Byte t of the words of a quad's four lanes, in lane order (a 4 x 4 byte transpose).
__device__ __forceinline__ uint32_t quad_plane(uint32_t x, int t) {
  x = __byte_perm(x, __shfl_xor_sync(0xffffffffu, x, 2), (t & 2) ? 0x3276 : 0x5410);
  return __byte_perm(x, __shfl_xor_sync(0xffffffffu, x, 1), (t & 1) ? 0x3715 : 0x6240);
}

// Code word `t` of every 32-dim group of a slot's row in shared memory.  Rows
// of 64 and 256 dims are 32 and 128 bytes apart, so lanes of different slots
// (g) start at different groups and sort the words afterwards: no two lanes
// of a load meet in a bank.
template <int HD>
__device__ __forceinline__ void key_words(const uint32_t* row, int g, int t, uint32_t (&w)[Q4Shape<HD>::G]) {
  if constexpr (HD == 16) {
    w[0] = t < 2 ? row[t] : 0u;
  } else if constexpr (HD == 64) {
    const int first = g >> 2;
    const uint32_t a = row[4 * first + t], b = row[4 * (first ^ 1) + t];
    w[0] = first ? b : a;
    w[1] = first ? a : b;
  } else {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = row[4 * ((i + g) & 7) + t];  // group (i + g) & 7
#pragma unroll
    for (int sh = 1; sh < 8; sh <<= 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = (g & sh) ? u[(i - sh) & 7] : u[i];
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = w[i];
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(THREADS) attend_q4_kernel(const AttendArgs a) {
  using S = Q4Shape<HD>;
  extern __shared__ __align__(128) uint8_t dyn[];
  int32_t* const logits = reinterpret_cast<int32_t*>(dyn + S::STAGES * S::STAGE_BYTES);
  __shared__ uint64_t full[S::STAGES], empty[S::STAGES];
  __shared__ int16_t lut[256];
  __shared__ int16_t s_q[HD];
  __shared__ uint64_t exchanged[2];  // the cluster's maxima and sums are here
  __shared__ int s_max[MAX_CLUSTER], s_redi[WARPS];
  __shared__ unsigned long long s_sum[MAX_CLUSTER], s_red[WARPS];
  __shared__ unsigned long long s_ctx[HD];
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], WARPS);
    }
    mbar_init(&exchanged[0], (uint32_t)parts);
    mbar_init(&exchanged[1], (uint32_t)parts);
    fence_barrier_init();
  }
  for (int i = tid; i < 256; i += THREADS) lut[i] = d_exp2_lut[i];
  if (tid < HD) s_ctx[tid] = 0;
  griddep_wait();
  griddep_launch();
  const long long bh = blockIdx.x / parts;
  const int h = (int)(bh % (long long)a.c.heads);
  const long long b = bh / (long long)a.c.heads;
  const long long len = (long long)a.lens[b] + a.len_offset;
  if (len <= 0 || len > (long long)a.c.capacity) {  // the same for the whole cluster
    if (tid == 0) nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
    return;
  }
  const int share = ((int)((len + parts - 1) / parts) + SHARE_UNIT - 1) / SHARE_UNIT * SHARE_UNIT;
  const long long first = (long long)part * share;
  const int n = (int)max(0ll, min((long long)share, len - first));
  const size_t slot0 = (size_t)bh * a.c.capacity + (size_t)first;
  if (tid < HD) s_q[tid] = a.q[b * a.ldq + (long long)h * HD + tid];
  cluster.sync();  // every CTA's barriers are ready
  const int tiles = (n + S::TILE - 1) / S::TILE;

  if (warp == WARPS) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      int issued = 0;
      for (int it = 0; it < 2 * tiles; ++it) {
        const int s = it % S::STAGES;
        if (it >= S::STAGES && !mbar_wait(&empty[s], ((it / S::STAGES) - 1) & 1, a.st)) break;
        const bool value = it >= tiles;
        const int at = (value ? it - tiles : it) * S::TILE;
        // whole 16-slot runs: a multiple of 16 bytes, and inside the capacity
        const uint32_t slots = (uint32_t)(min(S::TILE, n - at) + 15) & ~15u;
        uint8_t* stage = dyn + s * S::STAGE_BYTES;
        mbar_arrive_expect_tx(&full[s], slots * (HD / 2 + 4 * S::G));
        bulk_load(stage, (value ? a.c.v_codes : a.c.k_codes) + (slot0 + at) * (HD / 2), slots * (HD / 2), &full[s]);
        bulk_load(stage + S::CODE_BYTES, (value ? a.c.v_scales : a.c.k_scales) + (slot0 + at) * S::G, slots * 4 * S::G,
                  &full[s]);
        issued = it + 1;
      }
      for (int it = (issued > S::STAGES ? issued - S::STAGES : 0); it < issued; ++it)
        mbar_wait(&full[it % S::STAGES], (it / S::STAGES) & 1, a.st);
    }
    __syncwarp();
    cluster.sync();
    cluster.sync();
    return;
  }

  // -------------------------------------------------------------------- keys
  const int g = lane >> 2, t = lane & 3;
  // B fragments of group c: columns 4 (c & 1) + {0: h, 1: l, 2: ones}; k index
  // 4 t + i holds dim 8 t + 2 i of the group, 16 + 4 t + i dim 8 t + 2 i + 1.
  uint32_t qb[S::G][2];
  int qsum[S::PAIRS];  // sum of q over group 2 i + (t >> 1), on the lanes of its column 0
#pragma unroll
  for (int i = 0; i < S::PAIRS; ++i) qsum[i] = 0;
#pragma unroll
  for (int c = 0; c < S::G; ++c) {
    const int role = g - 4 * (c & 1);
    int sum = 0;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int dim = 8 * t + 2 * i + o;
        const int q = dim < HD ? (int)s_q[(32 * c + dim) % HD] : 0;
        sum += q;
        const int byte = role == 0 ? q >> 8 : role == 1 ? (q & 255) - 128 : role == 2 ? 1 : 0;
        w |= (uint32_t)(byte & 255) << (8 * i);
      }
      qb[c][o] = w;
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (t == 2 * (c & 1)) qsum[c / 2] = sum;
  }
  // a lane's part of a group's dot: 256 h + l on its columns 0 and 1, 128 times the codes' sum on column 2
  const int alpha = (t & 1) ? 128 : 256, beta = (t & 1) ? 0 : 1;
  const int group = S::G == 1 ? 0 : t >> 1;  // of a pair

  bool bad = false, alive = true;
  int mx = INT_MIN;
  for (int it = 0; it < tiles && alive; ++it) {
    const int s = it % S::STAGES;
    alive = mbar_wait(&full[s], (it / S::STAGES) & 1, a.st);
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(dyn + s * S::STAGE_BYTES);
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(dyn + s * S::STAGE_BYTES + S::CODE_BYTES);
    const int left = n - it * S::TILE;
    // 16 slots from r: lanes t even end with slot g's part of group t >> 1, odd ones with slot g + 8's
    auto dots = [&](int r) -> long long {
      uint32_t w0[S::G], w1[S::G];
      key_words<HD>(codes + (r + g) * S::WORDS, g, t, w0);
      key_words<HD>(codes + (r + g + 8) * S::WORDS, g, t, w1);
      long long v0 = 0, v1 = 0;
#pragma unroll
      for (int p = 0; p < S::PAIRS; ++p) {
        int c[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 2 * p; j < 2 * p + 2 && j < S::G; ++j) {
          const uint32_t frag[4] = {w0[j] & LOW, w1[j] & LOW, (w0[j] >> 4) & LOW, (w1[j] >> 4) & LOW};
          mma_u8s8(c, frag, qb[j]);
        }
        const uint32_t s0 = scales[(r + g) * S::G + 2 * p + group], s1 = scales[(r + g + 8) * S::G + 2 * p + group];
        v0 += (long long)(alpha * c[0] + beta * c[1]) * (int)(s0 & 0xFFFF) + (long long)qsum[p] * ((int)s0 >> 16);
        v1 += (long long)(alpha * c[2] + beta * c[3]) * (int)(s1 & 0xFFFF) + (long long)qsum[p] * ((int)s1 >> 16);
      }
      const long long keep = (t & 1) ? v1 : v0;
      return keep + __shfl_xor_sync(0xffffffffu, (t & 1) ? v0 : v1, 1);
    };
#pragma unroll
    for (int u = 0; u < S::TILE; u += WARPS * S::UNIT) {
      const int r = u + S::UNIT * warp;
      if (r >= left) break;
      int slot = r + g + 8 * (t & 1);
      bool live = true;
      long long v = dots(r);
      if constexpr (S::UNIT == 32) {  // lanes t >= 2 finish the second 16 slots
        const long long w = dots(r + 16);
        v = ((t & 2) ? w : v) + __shfl_xor_sync(0xffffffffu, (t & 2) ? v : w, 2);
        slot += 8 * (t & 2);
      } else {
        v += __shfl_xor_sync(0xffffffffu, v, 2);
        live = t < 2;
      }
      if (live && slot < left) {
        const long long lg = v >> S::SHIFT;
        bad = bad || lg != (long long)(int)lg;
        logits[it * S::TILE + slot] = (int)lg;
        mx = max(mx, (int)lg);  // MASKED_LOGIT is INT_MIN: it never raises the maximum
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
  }
  if (bad) nsrl_flag(a.st, NSRL_FLAG_LOGIT_RANGE);
  mx = __reduce_max_sync(0xffffffffu, mx);
  if (lane == 0) s_redi[warp] = mx;
  consumers_sync();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) mx = max(mx, s_redi[w]);
  alive = exchange(cluster, s_max, &exchanged[0], mx, part, parts, a.st) && alive;
  for (int r = 0; r < parts; ++r) mx = max(mx, s_max[r]);
  const bool any = mx != INT_MIN;
  if (!any && tid == 0 && part == 0) nsrl_flag(a.st, NSRL_FLAG_ALL_MASKED);

  // ---------------------------------------------------------------- softmax
  unsigned long long sum = 0;
#pragma unroll 4
  for (int j = tid; j < n; j += CONSUMERS) {
    const int lg = logits[j];
    // exp2_neg_q15 of lg - mx <= 0, whose magnitude fits 32 bits
    const unsigned mag = (unsigned)mx - (unsigned)lg;
    const int w = lg == INT_MIN || mag >= 15u * 256u ? 0 : (int)lut[mag & 255] >> (mag >> 8);
    logits[j] = w;
    sum += (unsigned)w;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_red[warp] = sum;
  consumers_sync();
  sum = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) sum += s_red[w];
  alive = exchange(cluster, s_sum, &exchanged[1], sum, part, parts, a.st) && alive;
  sum = 0;
  for (int r = 0; r < parts; ++r) sum += s_sum[r];
  // The slot at the maximum has weight 32767, so sum >= 32767, inv <= 65793 and
  // w inv + 2^15 < 2^32: sat_i16(rhu64(w * inv, 16)) in 32 bits.
  const unsigned inv = any ? recip_sum_q31(sum) : 0u;
  const int padded = (n + SHARE_UNIT - 1) / SHARE_UNIT * SHARE_UNIT;
  int32_t* const scores = a.c.scores ? a.c.scores + slot0 : nullptr;
#pragma unroll 4
  for (int j = tid; j < padded; j += CONSUMERS) {
    if (j >= n) {
      logits[j] = 0;  // slots of the last value MMA past the share weigh nothing
    } else {
      const int p = (int)min(((unsigned)logits[j] * inv + 32768u) >> 16, 32767u);
      logits[j] = p;
      if (scores) scores[j] = add_sat(scores[j], p);
    }
  }
  consumers_sync();

  // ------------------------------------------------------------------ values
  // A warp's unit is 32 slots of one pair of groups (64 dims).  Lane (g, t)
  // reads code word g of the pair for slots 4 j + t; byte i of it holds dims
  // 2 i and 2 i + 1, rows g and g + 8 of MMA i (16 dims a head: byte g, MMA 0).
  // High halves are left in place (16 times the code: rows g + 8 shift down at
  // the end).  The weights p scale are formed once per slot and group, on lane
  // 4 (slot & 3 | slot >> 4 & 1 << 2) + (slot >> 2 & 3), and their byte planes
  // handed to the lanes of their column.
  constexpr int MMAS = HD == 16 ? 1 : 4;
  const int pair = warp % S::PAIRS;
  int acc[MMAS][4];
#pragma unroll
  for (int i = 0; i < MMAS; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0;
  long long zero_part[2] = {0, 0};  // sum of p zero over this lane's slots, per group of the pair
  const int own = 4 * t + (g & 3) + 16 * (g >> 2);  // the slot whose weights this lane forms
  const int from = 4 * t + (g & 3);                 // the lane with plane g & 3 of slots 4 i + t
  const uint32_t byte2 = (uint32_t)(g & 3) | ((uint32_t)((g & 3) + 4) << 4);  // byte g & 3 of two words
  for (int it = tiles; it < 2 * tiles && alive; ++it) {
    const int s = it % S::STAGES;
    alive = mbar_wait(&full[s], (it / S::STAGES) & 1, a.st);
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(dyn + s * S::STAGE_BYTES);
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(dyn + s * S::STAGE_BYTES + S::CODE_BYTES);
    const int at = (it - tiles) * S::TILE, left = n - at;
#pragma unroll
    for (int u = 0; u < S::TILE / 32; u += WARPS / S::PAIRS) {
      const int r = 32 * (u + warp / S::PAIRS);
      if (r >= left) break;
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = codes[(r + 4 * j + t) * S::WORDS + (HD == 16 ? g >> 2 : 8 * pair + g)];
      const int p = logits[at + r + own];
      uint32_t bf[2];
      if constexpr (HD == 16) {
        const uint32_t sw = scales[r + own];
        zero_part[0] += (long long)p * ((int)sw >> 16);
        const uint32_t plane = quad_plane((uint32_t)p * (sw & 0xFFFF), t);
        bf[0] = __shfl_sync(0xffffffffu, plane, from);
        bf[1] = __shfl_sync(0xffffffffu, plane, from + 16);
      } else {
        const uint2 sw = *reinterpret_cast<const uint2*>(scales + (r + own) * S::G + 2 * pair);
        zero_part[0] += (long long)p * ((int)sw.x >> 16);
        zero_part[1] += (long long)p * ((int)sw.y >> 16);
        const uint32_t plane0 = quad_plane((uint32_t)p * (sw.x & 0xFFFF), t);
        const uint32_t plane1 = quad_plane((uint32_t)p * (sw.y & 0xFFFF), t);
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const uint32_t x = __shfl_sync(0xffffffffu, plane0, from + 16 * o);
          const uint32_t y = __shfl_sync(0xffffffffu, plane1, from + 16 * o);
          bf[o] = (g >> 2) ? y : x;
        }
      }
      uint32_t by[2][MMAS];  // byte i of four slots' words
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const uint32_t* x = w + 4 * o;
        if constexpr (HD == 16) {
          by[o][0] = __byte_perm(__byte_perm(x[0], x[1], byte2), __byte_perm(x[2], x[3], byte2), 0x5410);
        } else {
          const uint32_t lo01 = __byte_perm(x[0], x[1], 0x5140), hi01 = __byte_perm(x[0], x[1], 0x7362);
          const uint32_t lo23 = __byte_perm(x[2], x[3], 0x5140), hi23 = __byte_perm(x[2], x[3], 0x7362);
          by[o][0] = __byte_perm(lo01, lo23, 0x5410);
          by[o][1] = __byte_perm(lo01, lo23, 0x7632);
          by[o][2] = __byte_perm(hi01, hi23, 0x5410);
          by[o][3] = __byte_perm(hi01, hi23, 0x7632);
        }
      }
#pragma unroll
      for (int i = 0; i < MMAS; ++i) {
        const uint32_t frag[4] = {by[0][i] & LOW, by[0][i] & HIGH, by[1][i] & LOW, by[1][i] & HIGH};
        mma_u8u8(acc[i], frag, bf);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[s]);
  }
  // Columns 2 t and 2 t + 1 are planes 2 (t & 1) and 2 (t & 1) + 1 of the pair's
  // group t >> 1; the lane's dims are of group g >> 2 of the pair.  s32 is enough:
  // 240 * 255 a slot over at most 16,384 slots a warp.
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    zero_part[0] += __shfl_xor_sync(0xffffffffu, zero_part[0], o);
    if (HD != 16) zero_part[1] += __shfl_xor_sync(0xffffffffu, zero_part[1], o);
  }
  const long long zeros = HD != 16 && (g >> 2) ? zero_part[1] : zero_part[0];
  const bool mine = (t & 1) == 0 && (HD == 16 ? t == 0 : (t >> 1) == (g >> 2));
#pragma unroll
  for (int i = 0; i < MMAS; ++i)
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const int lo = acc[i][2 * o] >> (4 * o), hi = acc[i][2 * o + 1] >> (4 * o);
      long long v = ((long long)lo + ((long long)hi << 8)) << (16 * (t & 1));
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      const int dim = HD == 16 ? 2 * g + o : 64 * pair + 8 * g + 2 * i + o;
      if (mine) atomicAdd(&s_ctx[dim], (unsigned long long)(v + zeros));
    }
  cluster.sync();
  if (part == 0 && tid < HD) {
    unsigned long long tot = 0;
    for (int r = 0; r < parts; ++r) tot += cluster.map_shared_rank(s_ctx, r)[tid];
    a.ctx[b * (long long)(a.c.heads * HD) + (long long)h * HD + tid] = sat_i16(rhu64((long long)tot, 15));
  }
  cluster.sync();  // no CTA leaves while rank 0 reads its partial context
}

template <int HD>
cudaError_t launch_attend(const AttendArgs& a, int parts, size_t share, cudaStream_t s) {
  const size_t smem = Q4Shape<HD>::STAGES * Q4Shape<HD>::STAGE_BYTES + share * sizeof(int32_t);
  cudaError_t e = cudaFuncSetAttribute(attend_q4_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.c.batch * a.c.heads * (size_t)parts));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, attend_q4_kernel<HD>, a);
}

}  // namespace

size_t q4_max_capacity() { return MAX_CLUSTER * MAX_SHARE; }

cudaError_t launch_attend_q4(const int16_t* q, size_t ldq, const nsrl_q4_cache& c, const int32_t* lens, int len_offset,
                             int16_t* ctx, nsrl_device_status* st, cudaStream_t s) {
  const size_t bh = c.batch * c.heads;
  if (bh == 0) return cudaSuccess;
  if (c.capacity > q4_max_capacity() || bh > 0x7fffffffull / MAX_CLUSTER) return cudaErrorInvalidValue;
  const AttendArgs a{c, q, (long long)ldq, lens, len_offset, ctx, st};
  int parts = 1;
  while (parts < MAX_CLUSTER &&
         ((c.capacity + parts - 1) / parts > MAX_SHARE || (bh * parts < 148 && c.capacity / parts >= 512)))
    parts *= 2;
  if (getenv("Q4PARTS")) parts = atoi(getenv("Q4PARTS"));
  const size_t share = ((c.capacity + parts - 1) / parts + SHARE_UNIT - 1) / SHARE_UNIT * SHARE_UNIT;
  const double slots = (double)bh * (double)c.capacity;
  ProfScope prof("attention_decode_q4", s, 4.0 * slots * (double)c.head_dim,
                 slots * ((double)c.head_dim + 8.0 * std::max<size_t>(1, c.head_dim / 32) + (c.scores ? 8.0 : 0.0)));
  const cudaError_t e = c.head_dim == 16   ? launch_attend<16>(a, parts, share, s)
                        : c.head_dim == 64 ? launch_attend<64>(a, parts, share, s)
                                           : launch_attend<256>(a, parts, share, s);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace nsrl
