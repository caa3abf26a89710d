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
// shared memory.  The cache is read once.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace cg = cooperative_groups;

namespace nsrl {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_CLUSTER = 8;
constexpr int SHARE_UNIT = 32;
constexpr size_t MAX_SHARE = 49152;  // logits of a CTA: 192 KB

struct AttendArgs {
  nsrl_q4_cache c;
  const int16_t* q;
  long long ldq;
  const int32_t* lens;
  int len_offset;
  int16_t* ctx;
  nsrl_device_status* st;
};

template <int HD>
__global__ void __launch_bounds__(THREADS) attend_q4_kernel(const AttendArgs a) {
  constexpr int LPK = HD / 8;  // lanes of a slot
  constexpr int LPG = HD < 32 ? HD / 8 : 4;
  constexpr int G = HD < 32 ? 1 : HD / 32;
  constexpr int SHIFT = HD == 16 ? 2 : HD == 64 ? 3 : 4;
  constexpr int SLOTS = THREADS / LPK;  // slots of a pass of the CTA
  extern __shared__ __align__(16) int32_t logits[];
  __shared__ int16_t lut[256];
  __shared__ long long s_max, s_red[WARPS];
  __shared__ unsigned long long s_sum;
  __shared__ long long s_ctx[HD];
  const cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
  for (int i = tid; i < 256; i += THREADS) lut[i] = d_exp2_lut[i];
  if (tid < HD) s_ctx[tid] = 0;

  // ---- logits ----
  const int sub = tid % LPK, grp = tid / LPK;
  int q[8], qsum = 0;
  {
    const int16_t* qp = a.q + b * a.ldq + (long long)h * HD + 8 * sub;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q[i] = qp[i];
      qsum += q[i];
    }
  }
  const uint32_t* kc = reinterpret_cast<const uint32_t*>(a.c.k_codes) + slot0 * LPK;
  const uint32_t* vc = reinterpret_cast<const uint32_t*>(a.c.v_codes) + slot0 * LPK;
  const uint32_t* ks = a.c.k_scales + slot0 * G;
  const uint32_t* vs = a.c.v_scales + slot0 * G;
  bool bad = false;
  long long mx = LLONG_MIN;
  for (int j0 = 0; j0 < n; j0 += SLOTS) {
    const int j = j0 + grp;
    long long dot = 0;
    if (j < n) {
      const uint32_t w = kc[(size_t)j * LPK + sub], sw = ks[(size_t)j * G + sub / LPG];
      int d = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) d += q[i] * (int)((w >> (4 * i)) & 15);
      dot = (long long)d * (int)(sw & 0xFFFF) + (long long)qsum * (int)(int16_t)(sw >> 16);
    }
#pragma unroll
    for (int o = 1; o < LPK; o <<= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (sub == 0 && j < n) {
      const long long lg = dot >> SHIFT;
      if (lg < INT_MIN || lg > INT_MAX) bad = true;
      logits[j] = (int32_t)lg;
      if ((int32_t)lg != INT_MIN) mx = max(mx, (long long)(int32_t)lg);  // MASKED_LOGIT is excluded from the max
    }
  }
  if (bad) nsrl_flag(a.st, NSRL_FLAG_LOGIT_RANGE);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) s_red[warp] = mx;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < WARPS; ++w) mx = max(mx, s_red[w]);
    s_max = mx;
  }
  cluster.sync();
  mx = LLONG_MIN;
  for (int r = 0; r < parts; ++r) mx = max(mx, *cluster.map_shared_rank(&s_max, r));
  const bool any = mx != LLONG_MIN;
  if (!any && tid == 0 && part == 0) nsrl_flag(a.st, NSRL_FLAG_ALL_MASKED);

  // ---- weights and their sum ----
  unsigned long long sum = 0;
  for (int j = tid; j < n; j += THREADS) {
    const int32_t lg = logits[j];
    const int w = !any || lg == INT_MIN ? 0 : exp2_neg_q15(lut, (long long)lg - mx);
    logits[j] = w;
    sum += (unsigned long long)w;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_red[warp] = (long long)sum;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < WARPS; ++w) sum += (unsigned long long)s_red[w];
    s_sum = sum;
  }
  cluster.sync();
  sum = 0;
  for (int r = 0; r < parts; ++r) sum += *cluster.map_shared_rank(&s_sum, r);
  const long long inv = any ? (long long)recip_sum_q31(sum) : 0;
  for (int j = tid; j < n; j += THREADS) {
    const int p = (int)sat_i16(rhu64((long long)logits[j] * inv, 16));
    logits[j] = p;
    if (a.c.scores) {
      const long long sc = (long long)a.c.scores[slot0 + j] + p;
      a.c.scores[slot0 + j] = (int32_t)min(sc, 2147483647ll);
    }
  }
  __syncthreads();

  // ---- context ----
  long long acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0;
  for (int j = grp; j < n; j += SLOTS) {
    const uint32_t w = vc[(size_t)j * LPK + sub], sw = vs[(size_t)j * G + sub / LPG];
    const long long p = logits[j];
    const int scale = (int)(sw & 0xFFFF), zero = (int)(int16_t)(sw >> 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += p * (zero + scale * (int)((w >> (4 * i)) & 15));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    atomicAdd(reinterpret_cast<unsigned long long*>(&s_ctx[8 * sub + i]), (unsigned long long)acc[i]);
  cluster.sync();
  if (part == 0 && tid < HD) {
    long long tot = 0;
    for (int r = 0; r < parts; ++r) tot += cluster.map_shared_rank(s_ctx, r)[tid];
    a.ctx[b * (long long)(a.c.heads * HD) + (long long)h * HD + tid] = sat_i16(rhu64(tot, 15));
  }
  cluster.sync();  // no CTA leaves while rank 0 reads its partial context
}

template <int HD>
cudaError_t launch_attend(const AttendArgs& a, int parts, size_t smem, cudaStream_t s) {
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
  const size_t share = ((c.capacity + parts - 1) / parts + SHARE_UNIT - 1) / SHARE_UNIT * SHARE_UNIT;
  const double slots = (double)bh * (double)c.capacity;
  ProfScope prof("attention_decode_q4", s, 4.0 * slots * (double)c.head_dim,
                 slots * ((double)c.head_dim + 8.0 * std::max<size_t>(1, c.head_dim / 32) + (c.scores ? 8.0 : 0.0)));
  const cudaError_t e = c.head_dim == 16   ? launch_attend<16>(a, parts, share * 4, s)
                        : c.head_dim == 64 ? launch_attend<64>(a, parts, share * 4, s)
                                           : launch_attend<256>(a, parts, share * 4, s);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace nsrl
