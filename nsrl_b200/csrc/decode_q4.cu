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
// Bound by memory (80 bytes a slot of 64 dims, 88 with scores) while an SM
// spends less than about 3.5 cycles on a slot, so instructions are counted:
//   keys:   a lane owns a slot; codes widen to bytes and meet the query's high
//           (signed) and low (unsigned) byte planes in dp4a, 32 a slot.
//   values: int8 MMAs (m16n8k32): A = 16 dims x 32 slots (a 4 x 4 byte
//           transpose by PRMT), B = the four byte planes of p_j scale_jg of two
//           groups, one column each.  An MMA takes 32 cycles of its quarter SM,
//           one cycle a slot in all; for the keys, whose products need no
//           transpose, dp4a costs fewer instructions.
// Everything is exact in s32 until it is combined in 64 bits.  Two warps
// stream tiles of codes and scales (K, then V) through a ring of bulk copies,
// so value tiles arrive while the softmax runs (waiting for a stage and
// refilling it takes a warp about 375 cycles whatever the size, more than a
// tile's share of the memory's time: hence two).  Teams of consumer warps take
// the tiles in turn, so that one team's latencies hide behind the others'.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace cg = cooperative_groups;

namespace nsrl {
namespace {

constexpr int WARPS = 16, COPIERS = 2;
constexpr int CONSUMERS = 32 * WARPS, THREADS = CONSUMERS + 32 * COPIERS;
constexpr int MAX_CLUSTER = 16;
constexpr int SHARE_UNIT = 32;       // slots of a value MMA
constexpr size_t MAX_SHARE = 32768;  // logits of a CTA: 128 KB

template <int HD>
struct Q4Shape {
  static constexpr int WORDS = HD / 8;             // code words of a slot
  static constexpr int G = HD < 32 ? 1 : HD / 32;  // groups
  static constexpr int GW = HD < 32 ? HD / 8 : 4;  // code words of a group
  static constexpr int PAIRS = (G + 1) / 2;        // pairs of groups, 64 dims each
  static constexpr int SHIFT = HD == 16 ? 2 : HD == 64 ? 3 : 4;
  static constexpr int TILE = HD == 16 ? 512 : HD == 64 ? 256 : 128;  // slots of a stage
  static constexpr int TEAM = HD == 256 ? 4 : 8;                      // warps that share a tile
  static constexpr int TEAMS = WARPS / TEAM;
  static constexpr int STAGES = 4;
  static constexpr int CODE_BYTES = TILE * HD / 2, SCALE_BYTES = TILE * G * 4;
  static constexpr int STAGE_BYTES = CODE_BYTES + SCALE_BYTES;
  static constexpr int Q_STRIDE = 4 * GW + 4;  // query words of a group in shared memory, padded against conflicts
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

__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0, %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(20000u)
      : "memory");
  return ok != 0;
}

// Gives `value` to slot `part` of every CTA of the cluster and waits (bounded)
// until all `parts` values are here.  All consumer threads call it with the
// same arguments; thread r serves rank r.
template <typename T>
__device__ __forceinline__ bool exchange(const cg::cluster_group& cluster, T* values, uint64_t* bar, T value, int part,
                                         int parts, nsrl_device_status* st) {
  if ((int)threadIdx.x < parts) {
    cluster.map_shared_rank(values, threadIdx.x)[part] = value;
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(bar)), "r"(threadIdx.x));
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
  }
  if (try_wait_cluster(bar)) return true;
  const unsigned long long t0 = global_ns();
  for (uint32_t i = 0;; ++i) {
    if (try_wait_cluster(bar)) return true;
    if ((i & 15u) == 15u && global_ns() - t0 > NSRL_WAIT_NS) {
      nsrl_flag(st, NSRL_FLAG_WAIT_TIMEOUT);
      return false;
    }
  }
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

template <int HD>
__global__ void __launch_bounds__(THREADS, HD == 256 ? 1 : 2) attend_q4_kernel(const AttendArgs a) {
  using S = Q4Shape<HD>;
  extern __shared__ __align__(128) uint8_t dyn[];
  int32_t* const logits = reinterpret_cast<int32_t*>(dyn + S::STAGES * S::STAGE_BYTES);
  __shared__ uint64_t full[S::STAGES], empty[S::STAGES];
  __shared__ uint64_t exchanged[2];  // the cluster's maxima and sums are here
  __shared__ int16_t lut[256];
  __shared__ uint32_t recip[128];
  // per group and code word {h of the even dims, h of the odd dims, l even, l odd}; then 16 times the group's sum of q
  __shared__ __align__(16) uint32_t s_q[S::G * S::Q_STRIDE];
  __shared__ int s_max[MAX_CLUSTER], s_redi[WARPS];
  __shared__ unsigned s_red[WARPS];
  __shared__ unsigned long long s_sum[MAX_CLUSTER];
  __shared__ long long s_part[WARPS / S::PAIRS][HD], s_ctx[HD];
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == CONSUMERS) {  // the copying warps do not wait for the others
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], S::TEAM);
    }
    mbar_init(&exchanged[0], (uint32_t)parts);
    mbar_init(&exchanged[1], (uint32_t)parts);
    fence_barrier_init();
  }
  if (tid < 256)
    lut[tid] = d_exp2_lut[tid];
  else if (tid < 256 + 128)
    recip[tid - 256] = d_recip_lut[tid - 256];
  griddep_wait();
  griddep_launch();
  const unsigned bh = blockIdx.x / (unsigned)parts;
  const unsigned b = bh / (unsigned)a.c.heads, h = bh - b * (unsigned)a.c.heads;
  int q8[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (tid < S::WORDS) {
    const int16_t* qp = a.q + b * a.ldq + (long long)h * HD + 8 * tid;
#pragma unroll
    for (int i = 0; i < 8; ++i) q8[i] = qp[i];
  }
  const long long len = (long long)a.lens[b] + a.len_offset;
  if (len <= 0 || len > (long long)a.c.capacity) {  // the same for the whole cluster
    if (tid == 0) nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
    return;
  }
  const int share = ((int)((len + parts - 1) / parts) + SHARE_UNIT - 1) / SHARE_UNIT * SHARE_UNIT;
  const long long first = (long long)part * share;
  const int n = (int)max(0ll, min((long long)share, len - first));
  const size_t slot0 = (size_t)bh * a.c.capacity + (size_t)first;
  const int tiles = (n + S::TILE - 1) / S::TILE;

  if (warp >= WARPS) {
    // ---------------------------------------------------------------- copies
    if (parts > 1) {
      cluster.sync();  // every CTA's barriers are ready
    } else {
      asm volatile("bar.sync 3, %0;" ::"n"(32 * COPIERS) : "memory");
      asm volatile("bar.arrive 2, %0;" ::"n"(THREADS) : "memory");
    }
    if (lane == 0) {
      static_assert(S::STAGES % COPIERS == 0);
      int issued = 0;
      for (int it = warp - WARPS; it < 2 * tiles; it += COPIERS) {
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
      // the copies in flight land before the CTA may leave: this warp's last ones, one a stage
      for (int it = issued - 1; it >= 0 && it > issued - 1 - S::STAGES; it -= COPIERS)
        mbar_wait(&full[it % S::STAGES], (it / S::STAGES) & 1, a.st);
    }
    __syncwarp();
    if (parts > 1) {
      cluster.sync();
      cluster.sync();
    }
    return;
  }

  if (tid < S::WORDS) {
    uint32_t w[4] = {0, 0, 0, 0};
    int sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum += q8[i];
      w[i & 1] |= (uint32_t)((q8[i] >> 8) & 255) << (8 * (i >> 1));
      w[2 + (i & 1)] |= (uint32_t)(q8[i] & 255) << (8 * (i >> 1));
    }
    const unsigned mask = S::WORDS >= 32 ? 0xffffffffu : (1u << S::WORDS) - 1;
#pragma unroll
    for (int o = 1; o < S::GW; o <<= 1) sum += __shfl_xor_sync(mask, sum, o);
    uint32_t* group = s_q + (tid / S::GW) * S::Q_STRIDE;
    *reinterpret_cast<uint4*>(group + 4 * (tid % S::GW)) = make_uint4(w[0], w[1], w[2], w[3]);
    if (tid % S::GW == 0) group[4 * S::GW] = (uint32_t)(16 * sum);
  }
  if (parts > 1)
    cluster.sync();
  else
    asm volatile("bar.sync 2, %0;" ::"n"(THREADS) : "memory");

  // -------------------------------------------------------------------- keys
  // A lane's slot is r + lane.  Lanes of 256-dim slots (128 bytes apart) start
  // at different groups, so that no two of a load meet in a bank.
  const int team = warp / S::TEAM, mate = warp % S::TEAM;
  constexpr bool HELD = S::G <= 2;  // the query's words in registers
  uint4 qw[HELD ? S::WORDS : 1];
  int qs[HELD ? S::G : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < S::G; ++i) qs[i] = (int)s_q[i * S::Q_STRIDE + 4 * S::GW];
#pragma unroll
    for (int i = 0; i < S::WORDS; ++i)
      qw[i] = *reinterpret_cast<const uint4*>(s_q + (i / S::GW) * S::Q_STRIDE + 4 * (i % S::GW));
  }
  bool bad = false, alive = true;
  int mx = INT_MIN;
  for (int it = team; it < tiles && alive; it += S::TEAMS) {
    const int s = it % S::STAGES;
    alive = mbar_wait(&full[s], (it / S::STAGES) & 1, a.st);
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(dyn + s * S::STAGE_BYTES);
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(dyn + s * S::STAGE_BYTES + S::CODE_BYTES);
    const int left = n - it * S::TILE;
    constexpr int UNITS = S::TILE / (32 * S::TEAM);
    // The rows go to registers first, where they fit, and the stage back to the copies.
    uint32_t held[HELD ? UNITS : 1][HELD ? S::WORDS : 1], held_scale[HELD ? UNITS : 1][HELD ? S::G : 1];
    if constexpr (HELD) {
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int slot = 32 * (u * S::TEAM + mate) + lane;
        const uint32_t* row = codes + slot * S::WORDS;
        if constexpr (HD == 16) {
          const uint2 x = *reinterpret_cast<const uint2*>(row);
          held[u][0] = x.x, held[u][1] = x.y;
          held_scale[u][0] = scales[slot];
        } else {
#pragma unroll
          for (int i = 0; i < S::WORDS; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(row + i);
            held[u][i] = x.x, held[u][i + 1] = x.y, held[u][i + 2] = x.z, held[u][i + 3] = x.w;
          }
          const uint2 x = *reinterpret_cast<const uint2*>(scales + 2 * slot);
          held_scale[u][0] = x.x, held_scale[u][1] = x.y;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int slot = 32 * (u * S::TEAM + mate) + lane;
      if (slot - lane >= left) break;
      long long v = 0;
#pragma unroll
      for (int i = 0; i < S::G; ++i) {
        const int c = HELD ? i : (i + lane) % S::G;
        uint32_t w[S::GW], sw;
        if constexpr (HELD) {
#pragma unroll
          for (int k = 0; k < S::GW; ++k) w[k] = held[u][S::GW * i + k];
          sw = held_scale[u][i];
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(codes + slot * S::WORDS + 4 * c);
          w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
          sw = scales[slot * S::G + c];
        }
        // odd dims stay in the high half bytes, 16 times over: the even dims' sums catch up
        int he = 0, ho = 0, le = 0, lo = 0;
#pragma unroll
        for (int k = 0; k < S::GW; ++k) {
          const uint4 q = HELD ? qw[S::GW * i + k] : *reinterpret_cast<const uint4*>(s_q + c * S::Q_STRIDE + 4 * k);
          he = dp4a_us(w[k] & LOW, q.x, he);
          ho = dp4a_us(w[k] & HIGH, q.y, ho);
          le = dp4a_uu(w[k] & LOW, q.z, le);
          lo = dp4a_uu(w[k] & HIGH, q.w, lo);
        }
        const int dot = (he * 256 + le) * 16 + (ho * 256 + lo);  // 16 sum q code, below 2^28
        const int qsum = HELD ? qs[i] : (int)s_q[c * S::Q_STRIDE + 4 * S::GW];
        v += (long long)dot * (int)(sw & 0xFFFF) + (long long)qsum * ((int)sw >> 16);
      }
      if (slot < left) {
        const long long lg = v >> (S::SHIFT + 4);
        bad = bad || lg != (long long)(int)lg;
        logits[it * S::TILE + slot] = (int)lg;
        mx = max(mx, (int)lg);  // MASKED_LOGIT is INT_MIN: it never raises the maximum
      }
    }
    if constexpr (!HELD) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
  }
  if (bad) nsrl_flag(a.st, NSRL_FLAG_LOGIT_RANGE);
  mx = __reduce_max_sync(0xffffffffu, mx);
  if (lane == 0) s_redi[warp] = mx;
  consumers_sync();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) mx = max(mx, s_redi[w]);
  if (parts > 1) {
    alive = exchange(cluster, s_max, &exchanged[0], mx, part, parts, a.st) && alive;
    for (int r = 0; r < parts; ++r) mx = max(mx, s_max[r]);
  }
  const bool any = mx != INT_MIN;
  if (!any && tid == 0 && part == 0) nsrl_flag(a.st, NSRL_FLAG_ALL_MASKED);

  // ---------------------------------------------------------------- softmax
  // Only the sum: the value pass weighs each slot again.  A CTA's sum is at most
  // 2^15 * MAX_SHARE = 2^30.
  unsigned part_sum = 0;
  const bool low = mx < INT_MIN + 15 * 256;  // MASKED_LOGIT would gather weight
  const int none = (int)((unsigned)mx - 15u * 256u);
#pragma unroll 2
  for (int j = 4 * tid; j < n; j += 4 * CONSUMERS) {
    int4 lg = *reinterpret_cast<const int4*>(logits + j);
    if (j + 3 >= n || low) {
      if (lg.x == INT_MIN) lg.x = none;
      if (lg.y == INT_MIN || j + 1 >= n) lg.y = none;
      if (lg.z == INT_MIN || j + 2 >= n) lg.z = none;
      if (lg.w == INT_MIN || j + 3 >= n) lg.w = none;
    }
    part_sum += weight(lut, lg.x, mx) + weight(lut, lg.y, mx) + weight(lut, lg.z, mx) + weight(lut, lg.w, mx);
  }
  part_sum = __reduce_add_sync(0xffffffffu, part_sum);
  if (lane == 0) s_red[warp] = part_sum;
  consumers_sync();
  unsigned long long sum = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) sum += s_red[w];
  if (parts > 1) {
    alive = exchange(cluster, s_sum, &exchanged[1], sum, part, parts, a.st) && alive;
    sum = 0;
    for (int r = 0; r < parts; ++r) sum += s_sum[r];
  }
  // The slot at the maximum has weight 32767, so sum >= 32767, inv <= 65793 and
  // w inv + 2^15 < 2^32: sat_i16(rhu64(w * inv, 16)) in 32 bits.
  unsigned inv = 0;
  if (any && sum >= 32767) {  // recip_sum_q31, the table in shared memory (the sum is smaller only after a timeout)
    const int shift = 63 - __clzll((long long)sum) - 7;
    inv = recip[((unsigned)(sum >> shift) & 255u) - 128] >> shift;
  }

  // ------------------------------------------------------------------ values
  // A warp's unit is 32 slots of one pair of groups (64 dims).  Transposing
  // matrix loads give lane (g, t) bytes 2 g and 2 g + 1 of a group's row for
  // slots 8 m + 2 t and 8 m + 2 t + 1; two loads and a PRMT make one byte of four
  // slots.  16 dims a head (8-byte rows): byte g of slots 4 j + t from words.  A
  // byte holds an even and an odd dim: row g of its MMA takes the byte as it is
  // (even + 16 odd), row g + 8 its high half (16 odd), and they part at the
  // end.  Slot `own` is this lane's to weigh (p, its score, p scale: 0 past the share); the
  // byte planes of p scale then go to the lanes of their column.
  constexpr int MMAS = HD == 16 ? 1 : 4;
  const int g = lane >> 2, t = lane & 3;
  const int pair = mate % S::PAIRS;
  int acc[MMAS][4];
#pragma unroll
  for (int i = 0; i < MMAS; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0;
  long long zero_part[2] = {0, 0};  // sum of p zero over this lane's slots, per group of the pair
  // The quad's slots are those of k = 4 (g & 3) + 16 (g >> 2) and the three after it.
  const int own = 16 * (g >> 2) + (HD == 16 ? 4 * t + (g & 3) : 8 * (t >> 1) + 2 * (g & 3) + (t & 1));
  const int from = 4 * t + (g & 3);  // the lane with plane g & 3 of the slots of k = 4 t; 16 further, of 16 + 4 t
  const uint32_t byte2 = (uint32_t)(g & 3) | ((uint32_t)((g & 3) + 4) << 4);  // byte g & 3 of two words
  int32_t* const scores = a.c.scores && pair == 0 ? a.c.scores + slot0 : nullptr;
  // A stage stays with one team for both passes, so that no wait skips a phase.
  static_assert(S::STAGES % S::TEAMS == 0);
  for (int it = tiles + (team - tiles % S::TEAMS + S::TEAMS) % S::TEAMS; it < 2 * tiles && alive; it += S::TEAMS) {
    const int s = it % S::STAGES;
    const int at = (it - tiles) * S::TILE, left = n - at;
    constexpr int STEP = S::TEAM / S::PAIRS, UNITS = S::TILE / 32 / STEP;
    int old[UNITS];
    if (scores) {
#pragma unroll
      for (int k = 0; k < UNITS; ++k) {
        const int slot = 32 * (k * STEP + mate / S::PAIRS) + own;
        old[k] = slot < left ? scores[at + slot] : 0;
      }
    }
    alive = mbar_wait(&full[s], (it / S::STAGES) & 1, a.st);
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(dyn + s * S::STAGE_BYTES);
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(dyn + s * S::STAGE_BYTES + S::CODE_BYTES);
    uint32_t w[UNITS][8];
    uint2 sw[UNITS];
    auto load = [&](int k) {
      const int r = 32 * (k * STEP + mate / S::PAIRS);
      if constexpr (HD == 16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[k][j] = codes[(r + 4 * j + t) * S::WORDS + (g >> 2)];
        sw[k] = make_uint2(scales[r + own], 0);
      } else {
        // lane l points at row r + l; w[k][4 e + m] is group e of slots 8 m ..
        const uint32_t row = smem_u32(codes + (r + lane) * S::WORDS + 8 * pair);
        load_matrices(row, w[k]);
        load_matrices(row + 16, w[k] + 4);
        sw[k] = *reinterpret_cast<const uint2*>(scales + (r + own) * S::G + 2 * pair);
      }
    };
    if constexpr (HD != 256) {
#pragma unroll
      for (int k = 0; k < UNITS; ++k) load(k);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
#pragma unroll
    for (int k = 0; k < UNITS; ++k) {
      const int r = 32 * (k * STEP + mate / S::PAIRS);
      if (r >= left) break;
      if constexpr (HD == 256) load(k);
      const int lg = logits[at + r + own];
      const bool masked = r + own >= left || lg == INT_MIN;
      const int p = masked ? 0 : (int)min((weight(lut, lg, mx) * inv + 32768u) >> 16, 32767u);
      if (scores && r + own < left) scores[at + r + own] = add_sat(old[k], p);
      uint32_t bf[2];
      zero_part[0] += (long long)p * ((int)sw[k].x >> 16);
      const uint32_t plane0 = quad_plane((uint32_t)p * (sw[k].x & 0xFFFF), t);
      if constexpr (HD == 16) {
        bf[0] = __shfl_sync(0xffffffffu, plane0, from);
        bf[1] = __shfl_sync(0xffffffffu, plane0, from + 16);
      } else {
        zero_part[1] += (long long)p * ((int)sw[k].y >> 16);
        const uint32_t plane1 = quad_plane((uint32_t)p * (sw[k].y & 0xFFFF), t);
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
          x = __byte_perm(__byte_perm(w[k][0], w[k][1], byte2), __byte_perm(w[k][2], w[k][3], byte2), 0x5410);
          y = __byte_perm(__byte_perm(w[k][4], w[k][5], byte2), __byte_perm(w[k][6], w[k][7], byte2), 0x5410);
        } else {  // MMA i: byte i & 1 of group i >> 1
          const uint32_t* m = w[k] + 4 * (i >> 1);
          x = __byte_perm(m[0], m[1], (i & 1) ? 0x7531 : 0x6420);
          y = __byte_perm(m[2], m[3], (i & 1) ? 0x7531 : 0x6420);
        }
        const uint32_t frag[4] = {x, x & HIGH, y, y & HIGH};
        mma_u8u8(acc[i], frag, bf);
      }
    }
    if constexpr (HD == 256) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
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
      if (t == 2 * (i >> 1)) s_part[warp / S::PAIRS][dim] = v + zero_part[i >> 1];
    }
  consumers_sync();
  long long total = 0;
  if (tid < HD) {
#pragma unroll
    for (int w = 0; w < WARPS / S::PAIRS; ++w) total += s_part[w][tid];
    s_ctx[tid] = total;
  }
  if (parts > 1) {
    cluster.sync();
    if (part == 0 && tid < HD)
      for (int r = 1; r < parts; ++r) total += cluster.map_shared_rank(s_ctx, r)[tid];
  }
  if (part == 0 && tid < HD)
    a.ctx[b * (long long)(a.c.heads * HD) + (long long)h * HD + tid] = sat_i16(rhu64(total, 15));
  if (parts > 1) cluster.sync();  // no CTA leaves while rank 0 reads its partial context
}

template <int HD>
cudaError_t launch_attend(const AttendArgs& a, int parts, size_t share, cudaStream_t s) {
  const size_t smem = Q4Shape<HD>::STAGES * Q4Shape<HD>::STAGE_BYTES + share * sizeof(int32_t);
  constexpr int MOST = Q4Shape<HD>::STAGES * Q4Shape<HD>::STAGE_BYTES + (int)MAX_SHARE * 4;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem((const void*)attend_q4_kernel<HD>, MOST, done);
  if (e == cudaSuccess && parts > 8)
    e = cudaFuncSetAttribute(attend_q4_kernel<HD>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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
  cfg.numAttrs = parts > 1 ? 2 : 1;  // a cluster of one would be packed two to an SM while others idle
  return cudaLaunchKernelEx(&cfg, attend_q4_kernel<HD>, a);
}

}  // namespace

size_t q4_max_capacity() { return 8 * MAX_SHARE; }

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
