// The 4-bit KV cache: append (quantise), read (dequantise) and eviction by
// accumulated attention weight.  The format is described in nsrl_b200.h.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace nsrl {
namespace {

constexpr int THREADS = 256;

// ---------------------------------------------------------- append, read ---
// A thread owns 8 dims of one (sequence, head, token), of the key and of the
// value: a 16-byte int16 access and a 4-byte code access each.  Threads run
// over dims, then tokens, then heads, so a warp's cache rows are contiguous
// and its int16 rows are whole 32-byte sectors (64 dims: 128 bytes a row).
// Bound by memory: 4 hd bytes of int16 and hd + 16 ceil(hd / 32) / 2 of cache
// per slot, against some 8 instructions an element.
struct AppendArgs {
  nsrl_q4_cache c;
  const int16_t* k;
  const int16_t* v;
  long long ld;
  long long tokens;
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

// Eight dims to eight codes; scale_word is the group's (LPG lanes of the warp).
template <int LPG>
__device__ __forceinline__ uint32_t quantise8(const uint4& u, uint32_t& scale_word) {
  int x[8];
  unpack8(u, x);
  int lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min(lo, x[i]);
    hi = max(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o < LPG; o <<= 1) {
    lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const unsigned scale = max(1u, (unsigned)(hi - lo + 14) / 15u);
  // floor(n / d) = n * ceil(2^32 / d) >> 32 while n d < 2^32 (Granlund and
  // Montgomery): n = 2 (x - lo) + scale < 2^17.1, d = 2 scale < 2^13.1
  const unsigned d = 2 * scale;
  const unsigned magic = 0xFFFFFFFFu / d + 1;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    int q = (int)__umulhi(2u * (unsigned)(x[i] - lo) + scale, magic);
    q -= lo + (int)scale * q > 32767 ? 1 : 0;
    codes |= (uint32_t)q << (4 * i);
  }
  scale_word = scale | ((uint32_t)lo << 16);
  return codes;
}

template <int HD>
__global__ void __launch_bounds__(THREADS) q4_append_kernel(const AppendArgs a, const bool vec) {
  constexpr int LPR = HD / 8;                // lanes of a row
  constexpr int LPG = HD < 32 ? HD / 8 : 4;  // lanes of a group
  constexpr int G = HD < 32 ? 1 : HD / 32;
  griddep_wait();
  griddep_launch();
  const long long total = (long long)a.c.batch * a.c.heads * a.tokens * LPR;
  const long long i = (long long)blockIdx.x * THREADS + threadIdx.x;
  const bool inside = i < total;  // every lane of a warp takes part in the shuffles
  const int sub = (int)(i % LPR);
  const long long row = i / LPR;
  const long long bh = inside ? row / a.tokens : 0;
  const long long t = row - bh * a.tokens;
  const int h = (int)(bh % (long long)a.c.heads);
  const long long b = bh / (long long)a.c.heads;
  const long long start = a.starts[b], count = a.counts ? (long long)a.counts[b] : a.tokens;
  const bool fits = start >= 0 && count >= 0 && count <= a.tokens && start + count <= (long long)a.c.capacity;
  if (inside && !fits && t == 0 && sub == 0 && h == 0) nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
  const bool live = inside && fits && t < count;
  uint4 uk = make_uint4(0, 0, 0, 0), uv = uk;
  if (live) {
    const long long off = (b * a.tokens + t) * a.ld + (long long)h * HD + 8 * sub;
    uk = load8(a.k + off, vec);
    uv = load8(a.v + off, vec);
  }
  uint32_t sk, sv;
  const uint32_t ck = quantise8<LPG>(uk, sk), cv = quantise8<LPG>(uv, sv);
  if (!live) return;
  const size_t slot = (size_t)bh * a.c.capacity + (size_t)(start + t);
  reinterpret_cast<uint32_t*>(a.c.k_codes)[slot * LPR + sub] = ck;
  reinterpret_cast<uint32_t*>(a.c.v_codes)[slot * LPR + sub] = cv;
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

template <int HD>
__global__ void __launch_bounds__(THREADS) q4_read_kernel(const ReadArgs a) {
  constexpr int LPR = HD / 8;
  constexpr int LPG = HD < 32 ? HD / 8 : 4;
  constexpr int G = HD < 32 ? 1 : HD / 32;
  griddep_wait();
  griddep_launch();
  const long long total = (long long)a.c.batch * a.c.heads * a.tokens * LPR;
  const long long i = (long long)blockIdx.x * THREADS + threadIdx.x;
  if (i >= total) return;
  const int sub = (int)(i % LPR);
  const long long row = i / LPR;
  const long long bh = row / a.tokens, t = row - bh * a.tokens;
  const long long b = bh / (long long)a.c.heads;
  const long long start = a.starts ? (long long)a.starts[b] : 0;
  if (start < 0 || start + a.tokens > (long long)a.c.capacity) {
    if (t == 0 && sub == 0) nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
    return;
  }
  const size_t slot = (size_t)bh * a.c.capacity + (size_t)(start + t);
  const uint32_t ck = reinterpret_cast<const uint32_t*>(a.c.k_codes)[slot * LPR + sub];
  const uint32_t cv = reinterpret_cast<const uint32_t*>(a.c.v_codes)[slot * LPR + sub];
  const uint32_t sk = a.c.k_scales[slot * G + sub / LPG], sv = a.c.v_scales[slot * G + sub / LPG];
  reinterpret_cast<uint4*>(a.k)[i] = dequantise8(ck, sk);
  reinterpret_cast<uint4*>(a.v)[i] = dequantise8(cv, sv);
}

// ------------------------------------------------------------- eviction ----
// Two launches.  q4_select_kernel (one CTA per (sequence, head)) finds the
// keep-th largest key by radix selection, 8 bits a pass, where key =
// 2^31 for a protected slot, else max(score, 0); marks the kept slots (ties to
// the lower slot) in a shared-memory bitmap; lists the holes below `keep` and
// the kept slots at or past it, both in ascending order and equally many.
// q4_move_kernel copies the m-th listed slot into the m-th hole.  Sources lie
// at or past `keep` and destinations below it, so the moves need no order.
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

constexpr int SEL_THREADS = 1024, SEL_WARPS = SEL_THREADS / 32;

__global__ void __launch_bounds__(SEL_THREADS) q4_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t bitmap[];  // kept slots, [capacity / 32 + 1]
  __shared__ int hist[256];
  __shared__ int warp_a[SEL_WARPS], warp_b[SEL_WARPS];
  __shared__ unsigned s_prefix;
  __shared__ int s_want;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_wait();
  griddep_launch();
  const long long bh = blockIdx.x;
  const long long b = bh / (long long)a.c.heads;
  const int keep = (int)a.keep;
  const int n = a.lens[b];
  if (n < 0 || n > (int)a.c.capacity) {
    if (tid == 0) {
      nsrl_flag(a.st, NSRL_FLAG_BAD_LENGTH);
      a.moves[bh] = 0;
    }
    return;
  }
  const int32_t* scores = a.c.scores + bh * (long long)a.c.capacity;
  const int32_t* positions = a.c.positions + bh * (long long)a.c.capacity;
  int32_t* scores_out = a.scores_out + bh * (long long)a.c.capacity;
  int32_t* positions_out = a.positions_out + bh * (long long)a.c.capacity;
  const long long border = (long long)a.next[b] - a.recent;
  auto key = [&](int i) -> unsigned {
    const long long p = positions[i];
    return p < a.sinks || p >= border ? 0x80000000u : (unsigned)max(scores[i], 0);
  };
  if (n <= keep) {
    for (int i = tid; i < n; i += SEL_THREADS) {
      scores_out[i] = scores[i];
      positions_out[i] = positions[i];
    }
    if (tid == 0) a.moves[bh] = 0;
    return;
  }
  // ---- the keep-th largest key ----
  unsigned prefix = 0;
  int want = keep;  // how many of the keys that share the prefix stay
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += SEL_THREADS) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += SEL_THREADS) {
      const unsigned k = key(i);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
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
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (before < want && before + own[j] >= want) {
          s_prefix = prefix | (unsigned)(255 - 8 * lane - j) << shift;
          s_want = want - before;
        }
        before += own[j];
      }
    }
    __syncthreads();
    prefix = s_prefix;
    want = s_want;
    __syncthreads();
  }
  const unsigned border_key = prefix;  // keys above it stay, and the first `want` slots that equal it

  // Each warp takes one contiguous span of slots, 32 at a time, so that ranks
  // follow the slot order.
  const int span = ((n + SEL_WARPS - 1) / SEL_WARPS + 31) / 32 * 32;
  const int lo = min(n, warp * span), hi = min(n, lo + span);
  auto prefix_of_warps = [&](int* mine) {  // exclusive prefix of warp counts; all threads
    __syncthreads();
    int s = 0;
    for (int w = 0; w < warp; ++w) s += mine[w];
    return s;
  };
  int equal = 0;
  for (int i = lo + lane; i - lane < hi; i += 32) equal += __popc(__ballot_sync(0xffffffffu, i < hi && key(i) == border_key));
  if (lane == 0) warp_a[warp] = equal;
  int rank = prefix_of_warps(warp_a);
  int holes = 0, late = 0;
  for (int i = lo + lane; i - lane < hi; i += 32) {
    const unsigned k = i < hi ? key(i) : 0u;
    const unsigned eq = __ballot_sync(0xffffffffu, i < hi && k == border_key);
    const bool kept = i < hi && (k > border_key || (k == border_key && rank + __popc(eq & ((1u << lane) - 1)) < want));
    rank += __popc(eq);
    const unsigned kept_bits = __ballot_sync(0xffffffffu, kept);
    holes += __popc(__ballot_sync(0xffffffffu, i < hi && i < keep && !kept));
    late += __popc(__ballot_sync(0xffffffffu, kept && i >= keep));
    if (lane == 0) bitmap[i >> 5] = kept_bits;  // spans are multiples of 32 slots
    if (kept && i < keep) {
      scores_out[i] = scores[i];
      positions_out[i] = positions[i];
    }
  }
  __syncthreads();
  if (lane == 0) {
    warp_a[warp] = holes;
    warp_b[warp] = late;
  }
  int hole_rank = prefix_of_warps(warp_a), late_rank = prefix_of_warps(warp_b);
  int2* list = a.list + bh * a.most;
  for (int i = lo + lane; i - lane < hi; i += 32) {
    const bool kept = (bitmap[i >> 5] >> lane) & 1;
    const bool hole = i < hi && i < keep && !kept, moves = i < hi && i >= keep && kept;
    const unsigned hb = __ballot_sync(0xffffffffu, hole), mb = __ballot_sync(0xffffffffu, moves);
    const unsigned below = (1u << lane) - 1;
    if (hole) list[hole_rank + __popc(hb & below)].y = i;
    if (moves) list[late_rank + __popc(mb & below)].x = i;
    hole_rank += __popc(hb);
    late_rank += __popc(mb);
  }
  if (tid == SEL_THREADS - 1) a.moves[bh] = late_rank;  // the last warp's running rank is the total
}

// One warp per move: the slot's codes, scales, score and position as 4-byte words.
__global__ void __launch_bounds__(THREADS) q4_move_kernel(const EvictArgs a) {
  griddep_wait();
  griddep_launch();
  const long long bh = blockIdx.x;
  const int moves = a.moves[bh];
  const int cw = (int)a.c.head_dim / 8, gw = a.c.head_dim < 32 ? 1 : (int)a.c.head_dim / 32;
  const int words = 2 * cw + 2 * gw + 2;
  const int lane = threadIdx.x & 31;
  const size_t base = (size_t)bh * a.c.capacity;
  uint32_t* kc = reinterpret_cast<uint32_t*>(a.c.k_codes);
  uint32_t* vc = reinterpret_cast<uint32_t*>(a.c.v_codes);
  for (int m = blockIdx.y * (THREADS / 32) + (threadIdx.x >> 5); m < moves; m += gridDim.y * (THREADS / 32)) {
    const int2 e = a.list[bh * a.most + m];
    const size_t from = base + (size_t)e.x, to = base + (size_t)e.y;
    for (int w = lane; w < words; w += 32) {
      if (w < cw)
        kc[to * cw + w] = kc[from * cw + w];
      else if (w < 2 * cw)
        vc[to * cw + w - cw] = vc[from * cw + w - cw];
      else if (w < 2 * cw + gw)
        a.c.k_scales[to * gw + w - 2 * cw] = a.c.k_scales[from * gw + w - 2 * cw];
      else if (w < 2 * cw + 2 * gw)
        a.c.v_scales[to * gw + w - 2 * cw - gw] = a.c.v_scales[from * gw + w - 2 * cw - gw];
      else if (w == words - 2)
        a.scores_out[to] = a.c.scores[from];
      else
        a.positions_out[to] = a.c.positions[from];
    }
  }
  // lens_out may be lens, so it changes only after the selection has read it
  if (blockIdx.y == 0 && bh % (long long)a.c.heads == 0 && threadIdx.x == 0) {
    const long long b = bh / (long long)a.c.heads;
    const int n = a.lens[b];
    if (n >= 0 && n <= (int)a.c.capacity) a.lens_out[b] = min(n, (int)a.keep);
  }
}

size_t most_moves(const nsrl_q4_cache& c, size_t keep) { return std::min(keep, c.capacity - keep); }
size_t list_offset(const nsrl_q4_cache& c) { return (c.batch * c.heads * sizeof(int32_t) + 255) & ~size_t(255); }

unsigned blocks_for(long long threads) { return (unsigned)((threads + THREADS - 1) / THREADS); }

}  // namespace

cudaError_t launch_q4_append(const nsrl_q4_cache& c, const int16_t* k, const int16_t* v, size_t ld, size_t tokens,
                             const int32_t* starts, const int32_t* counts, const int32_t* positions,
                             nsrl_device_status* st, cudaStream_t s) {
  const long long threads = (long long)(c.batch * c.heads * tokens * (c.head_dim / 8));
  if (threads == 0) return cudaSuccess;
  if (threads > (long long)THREADS * 0x7fffffffll) return cudaErrorInvalidValue;
  const AppendArgs a{c, k, v, (long long)ld, (long long)tokens, starts, counts, positions, st};
  const bool vec = ld % 8 == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
  const double rows = (double)(c.batch * c.heads) * (double)tokens;
  ProfScope prof("q4_append", s, 0.0, rows * (4.0 * c.head_dim + c.head_dim + 8.0 * std::max<size_t>(1, c.head_dim / 32)));
  auto* kernel = c.head_dim == 16 ? q4_append_kernel<16> : c.head_dim == 64 ? q4_append_kernel<64> : q4_append_kernel<256>;
  const cudaError_t e = launch_pdl(kernel, dim3(blocks_for(threads)), dim3(THREADS), 0, s, a, vec);
  return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_q4_read(const nsrl_q4_cache& c, const int32_t* starts, size_t tokens, int16_t* k, int16_t* v,
                           nsrl_device_status* st, cudaStream_t s) {
  const long long threads = (long long)(c.batch * c.heads * tokens * (c.head_dim / 8));
  if (threads == 0) return cudaSuccess;
  if (threads > (long long)THREADS * 0x7fffffffll) return cudaErrorInvalidValue;
  const ReadArgs a{c, starts, (long long)tokens, k, v, st};
  const double rows = (double)(c.batch * c.heads) * (double)tokens;
  ProfScope prof("q4_read", s, 0.0, rows * (4.0 * c.head_dim + c.head_dim + 8.0 * std::max<size_t>(1, c.head_dim / 32)));
  auto* kernel = c.head_dim == 16 ? q4_read_kernel<16> : c.head_dim == 64 ? q4_read_kernel<64> : q4_read_kernel<256>;
  const cudaError_t e = launch_pdl(kernel, dim3(blocks_for(threads)), dim3(THREADS), 0, s, a);
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
    ProfScope prof("q4_select", s, 0.0, 8.0 * (double)bh * (double)c.capacity);
    cudaError_t e = cudaFuncSetAttribute(q4_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = launch_pdl(q4_select_kernel, dim3((unsigned)bh), dim3(SEL_THREADS), smem, s, a);
    if (e != cudaSuccess) return e;
  }
  const unsigned chunks = (unsigned)std::max<size_t>(1, std::min<size_t>((a.most + 63) / 64, 64));
  ProfScope prof("q4_move", s, 0.0, 2.0 * (double)bh * (double)a.most * (double)c.head_dim);
  const cudaError_t e = launch_pdl(q4_move_kernel, dim3((unsigned)bh, chunks), dim3(THREADS), 0, s, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace nsrl
