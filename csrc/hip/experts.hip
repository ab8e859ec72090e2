// Routed experts: the router's top-k softmax, samples sorted by expert, and back with weights applied, with their
// gradients (raydp_amd/ops/expert_ops.py).
//
//   route     per row of logits z: the k largest (ties: lowest index), w_j = softmax over the chosen ones (renorm) or the
//             chosen entries of the softmax over all; backward with s = sum_j w_j dw_j:
//             renorm dz[chosen_j] = w_j (dw_j - s), else dz_e = [e chosen] w dw - p_e s
//   plan      a stable counting sort of the n = T k choices: row of each choice (position), choice of each row (source)
//   scatter   rows[position[t,j]] = (w[t,j]) x[t], rows without a choice 0; with h also dw[t,j] = <x[t], h[position[t,j]]>
//   gather    y[t] = sum_j (w[t,j]) rows[position[t,j]]
//
// scatter and gather are each other's gradients; every kernel works sample by sample, so that y crosses memory once, x and dy
// once for every four choices of a sample, the sums of a sample are one lane group's in a fixed order, and nothing needs
// atomics on floats.
#include "experts.h"
#include "rx_common.h"

namespace {

// ------------------------------------------------------------------------------------------------ element access
typedef u32x4 __attribute__((aligned(2))) u32x4_u;   // 16 bytes from any element (gfx950 reads unaligned vectors)

template <int DT> struct Elem;                       // 0 fp32, 1 bf16, 2 fp16
template <> struct Elem<0> {
  typedef float type;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<1> {
  typedef u16 type;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(u16 v) { return rx_bf2f(v); }
  static __device__ __forceinline__ u16 put(float v) { return rx_f2bf(v); }
};
template <> struct Elem<2> {
  typedef u16 type;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(u16 v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ u16 put(float v) { return __builtin_bit_cast(u16, (_Float16)v); }
};

template <int DT>
struct Vec {
  typedef typename Elem<DT>::type T;
  union {
    u32x4 w;
    T e[Elem<DT>::kVec];
  };
  // n: elements there (a row's last vector may be short); NT: streamed past the caches
  template <bool NT = false>
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= Elem<DT>::kVec) {
      if constexpr (NT) w = __builtin_nontemporal_load((const u32x4_u*)p);
      else w = *(const u32x4_u*)p;
    } else {
      w = (u32x4){0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < Elem<DT>::kVec - 1; ++i)
        if (i < n) e[i] = p[i];
    }
  }
  template <bool NT = false>
  __device__ __forceinline__ void store(T* p, int n) const {
    if (n >= Elem<DT>::kVec) {
      if constexpr (NT) __builtin_nontemporal_store(w, (u32x4_u*)p);
      else *(u32x4_u*)p = w;
    } else {
#pragma unroll
      for (int i = 0; i < Elem<DT>::kVec - 1; ++i)
        if (i < n) p[i] = e[i];
    }
  }
};

// ------------------------------------------------------------------------------------------------ router
// L lanes hold a row, V consecutive logits each, as keys that order as (logit, lowest index first) do and differ within a
// row. The next of the k largest keys is then one max per key and no bookkeeping of what was taken:
//   16-bit logits: (order-preserving 16 bits, 0xFFFF - index) in 32 bits, made two at a time. key - last wraps for every key
//                  below the last winner and so puts those above the ones taken: max over (key - last), two per v_max3.
//   fp32 logits:   (order-preserving 32 bits, 0xFFFF - index) as a positive double: one v_max_f64 for two words; a winner is
//                  struck out by its index.
// The order-preserving bits are the sign and magnitude as a number, shifted so that the magnitudes past infinity (NaN, of
// either sign) wrap to the bottom: the least key of a chosen logit is the first above minus infinity's, and -0 equals 0.
// A winner stays in its lane as the key; what it stands for is worked out afterwards.
typedef short rx_s16x2 __attribute__((ext_vector_type(2)));

template <int DT> struct Order;
template <> struct Order<0> {
  static constexpr uint32_t kInf = 0x7F800000u, kShift = 0x80000000u + 0x7FFFFFu, kLowest = 0xFFFFFFu;   // minus infinity's
};
template <> struct Order<1> {
  static constexpr uint32_t kInf = 0x7F80u, kShift = 0x8000u + 0x7Fu, kLowest = 0xFFu;
};
template <> struct Order<2> {
  static constexpr uint32_t kInf = 0x7C00u, kShift = 0x8000u + 0x3FFu, kLowest = 0x7FFu;
};

// of two 16-bit logits at once, and of an fp32 one
template <int DT>
__device__ __forceinline__ uint32_t order_pair(uint32_t x) {
  const rx_s16x2 v = __builtin_bit_cast(rx_s16x2, x), sign = v >> 15;
  const rx_s16x2 mag = v & (rx_s16x2){0x7FFF, 0x7FFF};
  constexpr short c = (short)Order<DT>::kShift;
  return __builtin_bit_cast(uint32_t, (rx_s16x2)(((mag ^ sign) - sign) + (rx_s16x2){c, c}));
}
__device__ __forceinline__ uint32_t order_one(uint32_t x) {
  const int sign = (int)x >> 31;
  return (uint32_t)((((int)(x & 0x7FFFFFFFu)) ^ sign) - sign) + Order<0>::kShift;
}
// the logit's bits again
template <int DT>
__device__ __forceinline__ float order_back(uint32_t o) {
  const uint32_t n = o - Order<DT>::kShift;                      // signed: the magnitude with the sign
  if constexpr (DT == 0) {
    const int sign = (int)n >> 31;
    return __uint_as_float((uint32_t)(((int)n ^ sign) - sign) | ((uint32_t)sign & 0x80000000u));
  } else {
    const int v = (int)(short)n, sign = v >> 31;
    return Elem<DT>::get((u16)(((v ^ sign) - sign) | (sign & 0x8000)));
  }
}

// LDS written by lanes of a wave is read by its other lanes after this
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Maxima and sums over groups of L lanes.
// (every lane has its partner: saying that none is read as anything else lets the move become part of the maximum)
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true));
}
template <int L>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  if constexpr (L >= 2) v = dpp_max<RX_DPP_XOR1>(v);
  if constexpr (L >= 4) v = dpp_max<RX_DPP_XOR2>(v);
  if constexpr (L >= 8) v = dpp_max<RX_DPP_HALF_MIRROR>(v);
  if constexpr (L >= 16) v = dpp_max<RX_DPP_MIRROR>(v);
  if constexpr (L >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(p[0], p[1]);
  }
  return v;
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (L >= 2) v += rx_dpp<RX_DPP_XOR1>(v);
  if constexpr (L >= 4) v += rx_dpp<RX_DPP_XOR2>(v);
  if constexpr (L >= 8) v += rx_dpp<RX_DPP_HALF_MIRROR>(v);
  if constexpr (L >= 16) v += rx_dpp<RX_DPP_MIRROR>(v);
  if constexpr (L >= 32) v += __shfl_xor(v, 16);
  if constexpr (L >= 64) v += __shfl_xor(v, 32);
  return v;
}
// (order in bits 61 to 30: the sign is 0 and the exponent never all ones)
__device__ __forceinline__ double as_key(uint32_t hi, uint32_t lo) {
  return __longlong_as_double((long long)(((unsigned long long)hi << 32) | lo));
}
// No key is a NaN, which fmax() has to allow for with a second instruction an operand (65536 x 256, k = 8: 29 us with it, 25
// without it). LAST: the result is moved across lanes next, which needs two wait states that the compiler does not see here.
template <bool LAST>
__device__ __forceinline__ double key_max(double a, double b) {
  double r;
  if constexpr (LAST) asm("v_max_f64 %0, %1, %2\n\ts_nop 1" : "=v"(r) : "v"(a), "v"(b));
  else asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
template <int CTRL>
__device__ __forceinline__ double dpp_key(double v) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(v);
  return __longlong_as_double((long long)(((unsigned long long)rx_dppu<CTRL>((uint32_t)(b >> 32)) << 32) | rx_dppu<CTRL>((uint32_t)b)));
}
template <int L>
__device__ __forceinline__ double group_max(double v) {
  if constexpr (L >= 2) v = key_max<true>(v, dpp_key<RX_DPP_XOR1>(v));
  if constexpr (L >= 4) v = key_max<true>(v, dpp_key<RX_DPP_XOR2>(v));
  if constexpr (L >= 8) v = key_max<true>(v, dpp_key<RX_DPP_HALF_MIRROR>(v));
  if constexpr (L >= 16) v = key_max<true>(v, dpp_key<RX_DPP_MIRROR>(v));
  if constexpr (L >= 32) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v);
    const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
    const auto l = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
    v = key_max<true>(as_key(h[0], l[0]), as_key(h[1], l[1]));
  }
  return v;
}

// e^x for x <= 0: relative error |x| 2^-24 and one ulp; 0 under 2^-126
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// Bound by instruction issue where k is large (65536 x 256, k = 8: 14 us in bf16, 22 in fp32, where reading takes 7 and 13),
// by memory where it is small (262144 x 64, k = 2: 9 us in bf16, 13 in fp32; reading takes 7 and 13).
template <int DT, int L, int V>
__global__ __launch_bounds__(256) void route_fwd_kernel(const typename Elem<DT>::type* __restrict__ z, long long ldz,
                                                        long long T, int E, int k, int renorm, float* __restrict__ w,
                                                        int* __restrict__ ids, float* __restrict__ norm) {
  constexpr int N = Elem<DT>::kVec;
  const int lane = threadIdx.x % L, first = lane * V;
  const long long t = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (t >= T) return;
  Vec<DT> x[V / N];
  if (E == L * V) {                         // (a power of two of them: nothing to look at per lane)
#pragma unroll
    for (int c = 0; c < V / N; ++c) x[c].load(z + t * ldz + first + c * N, N);
  } else {
    // places past the row are minus infinity with indexes past the row's: k <= E, so they are never taken
#pragma unroll
    for (int c = 0; c < V / N; ++c) {
      const int at = first + c * N;
      x[c].load(z + t * ldz + (at < E ? at : 0), E - at);
      if (at + N > E) {
#pragma unroll
        for (int q = 0; q < N; ++q)
          if (at + q >= E) x[c].e[q] = Elem<DT>::put(-__builtin_huge_valf());
      }
    }
  }
  // lane j % L keeps winner j: no more than kSlots of them
  constexpr int kSlots = V < kRouteMaxK / L ? V : L < kRouteMaxK ? kRouteMaxK / L : 1;
  uint32_t won[kSlots], at[kSlots];         // order, 0xFFFF - index (16 bits: both in won)
  uint32_t least = 0xFFFFFFFFu, top;        // a NaN's order is below minus infinity's; of the first winner
  if constexpr (DT == 0) {
    uint32_t hi[V], lo[V];
    const uint32_t low0 = 0xFFFFu - (uint32_t)first;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t o = order_one(__float_as_uint(x[i / N].e[i % N]));
      least = min(least, o);
      hi[i] = o >> 2;
      lo[i] = (o << 30) | (low0 - i);
    }
    const auto largest = [&] {
      double best = as_key(hi[0], lo[0]);
#pragma unroll
      for (int i = 1; i < V - 1; ++i) best = key_max<false>(best, as_key(hi[i], lo[i]));
      return (unsigned long long)__double_as_longlong(group_max<L>(key_max<true>(best, as_key(hi[V - 1], lo[V - 1]))));
    };
    unsigned long long last = largest();
    top = (uint32_t)(last >> 30);
    int j = 0;
#pragma unroll
    for (int r = 0; r < kSlots; ++r) {
      won[r] = at[r] = 0;
      for (int l = 0; l < L && j < k; ++l) {
        const uint32_t o = (uint32_t)(last >> 30), low = (uint32_t)last & 0xFFFFu;
        won[r] = lane == l ? o : won[r];
        at[r] = lane == l ? low : at[r];
        if (++j == k) break;
        // a winner loses its high word: what is left stands for less than minus infinity
        const uint32_t mine = low0 - low;
#pragma unroll
        for (int i = 0; i < V; ++i) hi[i] = mine == (uint32_t)i ? 0u : hi[i];
        last = largest();
      }
    }
  } else {
    uint32_t key[V];
    uint32_t low = 0xFFFFu - (uint32_t)first;
    low |= (low - 1) << 16;
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const uint32_t o = order_pair<DT>(x[i / N].w[(i % N) / 2]), lows = low - i * 0x10001u;
      key[i] = __builtin_amdgcn_perm(o, lows, 0x05040100u);        // (lower half of o, lower half of lows)
      key[i + 1] = __builtin_amdgcn_perm(o, lows, 0x07060302u);    // (the upper halves)
      least = min(least, min(key[i], key[i + 1]));
    }
    least >>= 16;
    uint32_t last = key[0];
#pragma unroll
    for (int i = 1; i < V; ++i) last = max(last, key[i]);
    last = group_max<L>(last);
    top = last >> 16;
    int j = 0;
#pragma unroll
    for (int r = 0; r < kSlots; ++r) {
      won[r] = 0;
      for (int l = 0; l < L && j < k; ++l) {
        won[r] = lane == l ? last : won[r];
        if (++j == k) break;
        uint32_t best = key[0] - last;
#pragma unroll
        for (int i = 1; i < V; ++i) best = max(best, key[i] - last);
        last += group_max<L>(best);
      }
    }
#pragma unroll
    for (int r = 0; r < kSlots; ++r) {
      at[r] = won[r] & 0xFFFFu;
      won[r] >>= 16;
    }
  }
  const float peak = top > Order<DT>::kLowest ? order_back<DT>(top) : 0.f;
  float part[kSlots], total = 0.f;
#pragma unroll
  for (int r = 0; r < kSlots; ++r) {
    part[r] = won[r] > Order<DT>::kLowest ? exp_neg(order_back<DT>(won[r]) - peak) : 0.f;     // (no winner: 0)
    total += part[r];
  }
  if (!renorm) {
    total = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) total += exp_neg(Elem<DT>::get(x[i / N].e[i % N]) - peak);
  }
  total = group_sum<L>(total);
  // a NaN in the row shows in all of its weights
  const unsigned long long rows = __ballot(least < Order<DT>::kLowest);
  const int shift = (threadIdx.x & 63) / L * L;
  const bool any = ((rows >> shift) & (L == 64 ? ~0ull : (1ull << (L & 63)) - 1)) != 0;
  const float inv = any ? __uint_as_float(0x7FC00000u) : total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;
#pragma unroll
  for (int r = 0; r < kSlots; ++r) {
    const int j = r * L + lane;
    if (j >= k) break;
    w[t * k + j] = part[r] * inv;
    ids[t * k + j] = won[r] > Order<DT>::kLowest ? (int)(0xFFFFu - at[r]) : -1;
  }
  if (norm != nullptr && lane == 0) {
    norm[2 * t] = peak;
    norm[2 * t + 1] = inv;
  }
}

// The chosen experts' terms are added through LDS, where a lane can reach any place of its row: in registers every one of
// the k would cost a comparison with every one of the V (65536 x 256 bf16, k = 8: 96 us that way, 16 this way; the bytes 13).
template <int DT, int L, int V>
__global__ __launch_bounds__(256) void route_bwd_kernel(const typename Elem<DT>::type* __restrict__ z, long long ldz,
                                                        const float* __restrict__ norm, const float* __restrict__ w,
                                                        const int* __restrict__ ids, const float* __restrict__ dw,
                                                        long long T, int E, int k,
                                                        typename Elem<DT>::type* __restrict__ dz) {
  __shared__ f32x4 rows[256 * V / 4 + 256 / L];      // 16 bytes between rows: their lanes then start on different banks
  constexpr int N = Elem<DT>::kVec;
  const int lane = threadIdx.x % L, first = lane * V;
  const long long t = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (t >= T) return;
  f32x4* row = rows + (threadIdx.x / L) * (L * V / 4 + 1);
  float s = 0.f;
  for (int j = lane; j < k; j += L)
    if (ids[t * k + j] >= 0) s = fmaf(w[t * k + j], dw[t * k + j], s);
  s = group_sum<L>(s);
  const bool full = norm != nullptr;
  const float peak = full ? norm[2 * t] : 0.f, scale = full ? -s * norm[2 * t + 1] : 0.f;
#pragma unroll
  for (int c = 0; c < V / N; ++c) {
    const int at = first + c * N;
    Vec<DT> x;
    if (full) x.load(z + t * ldz + (at < E ? at : 0), E - at);
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
      f32x4 g = {0.f, 0.f, 0.f, 0.f};
      if (full) {
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = scale * exp_neg(Elem<DT>::get(x.e[q * 4 + i]) - peak);
      }
      row[(at >> 2) + q] = g;
    }
  }
  wave_sync();
  float* flat = (float*)row;
  for (int j = lane; j < k; j += L) {
    const int e = ids[t * k + j];
    if (e >= 0) flat[e] += w[t * k + j] * (full ? dw[t * k + j] : dw[t * k + j] - s);
  }
  wave_sync();
#pragma unroll
  for (int c = 0; c < V / N; ++c) {
    const int at = first + c * N;
    Vec<DT> o;
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
      const f32x4 g = row[(at >> 2) + q];
#pragma unroll
      for (int i = 0; i < 4; ++i) o.e[q * 4 + i] = Elem<DT>::put(g[i]);
    }
    if (at < E) o.store(dz + t * E + at, E - at);
  }
}

// ------------------------------------------------------------------------------------------------ plan
constexpr int kPlanWaves = kPlanThreads / 64;

__device__ __forceinline__ int plan_expert(const void* ids, int wide, long long i, int E) {
  const long long e = wide ? ((const long long*)ids)[i] : (long long)((const int*)ids)[i];
  return e >= 0 && e < E ? (int)e : -1;
}

// counts[block][e] of a block's chunk of choices
__global__ __launch_bounds__(kPlanThreads) void plan_count_kernel(const void* __restrict__ ids, int wide, int n, int E,
                                                                  int chunk, int* __restrict__ counts) {
  __shared__ int hist[kMaxExperts];
  for (int e = threadIdx.x; e < E; e += kPlanThreads) hist[e] = 0;
  __syncthreads();
  const long long first = (long long)blockIdx.x * chunk;
  for (int c = threadIdx.x; c < chunk && first + c < n; c += kPlanThreads) {
    const int e = plan_expert(ids, wide, first + c, E);
    if (e >= 0) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kPlanThreads) counts[(long long)blockIdx.x * E + e] = hist[e];
}

// Bound by latency: 131072 choices among 64 experts take 4.8 us to count and 8 to rank, 4094 among 8 take 7.6 in one launch.
// Stable ranks. A workgroup's waves own consecutive pieces of its chunk; a wave takes 64 choices at a time, finds the
// lanes with the same expert by one ballot per bit of the expert's number, and counts on in LDS.
__global__ __launch_bounds__(kPlanThreads) void plan_rank_kernel(PlanArgs a) {
  extern __shared__ int lds[];
  int* total = lds;                         // [E] of all blocks, then the expert's first row
  int* before = total + kMaxExperts;        // [E] of the blocks before this one
  int* part = before + kMaxExperts;         // [16] scan
  int* next = part + kPlanWaves;            // [waves][E]: the next rank
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int E = a.E, piece = a.chunk / kPlanWaves;
  const long long first = (long long)blockIdx.x * a.chunk + (long long)wave * piece;
  for (int i = tid; i < E * kPlanWaves; i += kPlanThreads) next[i] = 0;
  for (int e = tid; e < E; e += kPlanThreads) total[e] = before[e] = 0;
  __syncthreads();
  for (int c = lane; c < piece && first + c < a.n; c += 64) {
    const int e = plan_expert(a.ids, a.wide, first + c, E);
    if (e >= 0) atomicAdd(&next[wave * E + e], 1);
  }
  if (a.counts != nullptr)
    for (int i = tid; i < a.blocks * E; i += kPlanThreads) {
      const int c = a.counts[i], b = i / E, e = i - b * E;
      if (c != 0) {
        atomicAdd(&total[e], c);
        if (b < (int)blockIdx.x) atomicAdd(&before[e], c);
      }
    }
  __syncthreads();
  int mine = 0;
  if (tid < E) {                            // (E <= threads)
    int at = before[tid];
    for (int w = 0; w < kPlanWaves; ++w) {
      const int c = next[w * E + tid];
      next[w * E + tid] = at;
      at += c;
    }
    mine = a.counts != nullptr ? total[tid] : at;
  }
  // exclusive sum over the experts
  int scan = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(scan, d);
    if (lane >= d) scan += o;
  }
  if (lane == 63) part[wave] = scan;
  __syncthreads();
  int base = 0, all = 0;
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w < wave) base += part[w];
    all += part[w];
  }
  const int start = a.capacity > 0 ? tid * a.capacity : base + scan - mine;
  if (tid < E) {
    total[tid] = start;
    if (blockIdx.x == 0) {
      a.load[tid] = mine;
      a.offsets[tid] = start;
    }
    if (a.capacity > 0) {                   // rows of an expert that no choice fills
      if (tid % (int)gridDim.x == (int)blockIdx.x) before[tid] = mine < a.capacity ? mine : a.capacity;
    }
  }
  if (tid == 0 && blockIdx.x == 0) a.offsets[E] = a.capacity > 0 ? E * a.capacity : all;
  __syncthreads();
  if (a.capacity > 0) {
    for (int e = blockIdx.x; e < E; e += gridDim.x)
      for (long long r = before[e] + tid; r < a.capacity; r += kPlanThreads) a.source[(long long)e * a.capacity + r] = -1;
  } else {
    for (long long r = (long long)all + blockIdx.x * kPlanThreads + tid; r < a.rows; r += (long long)gridDim.x * kPlanThreads)
      a.source[r] = -1;
  }
  int bits = 0;
  while ((1 << bits) < E) ++bits;
  int* mynext = next + wave * E;
  for (int c = 0; c < piece && first + c < a.n; c += 64) {
    const long long i = first + c + lane;
    const bool there = c + lane < piece && i < a.n;
    const int e = there ? plan_expert(a.ids, a.wide, i, E) : -1;
    unsigned long long same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long set = __ballot((e >> b) & 1);
      same &= ((e >> b) & 1) ? set : ~set;
    }
    int rank = 0, row = -1;
    if (e >= 0) {
      const int below = __popcll(same & ((1ull << lane) - 1));
      rank = mynext[e] + below;
      row = a.capacity > 0 && rank >= a.capacity ? -1 : total[e] + rank;
    }
    wave_sync();
    if (e >= 0 && (same >> lane) == 1ull) mynext[e] = rank + 1;     // the last of its lanes
    wave_sync();
    if (there) {
      a.position[i] = row;
      if (row >= 0) a.source[row] = (int)i;
    }
  }
}

// ------------------------------------------------------------------------------------------------ rows
// Both row kernels are bound by memory. A sample's row is 16 bytes a lane over as many lanes as it fills, at most a wave, and
// its expert rows are in flight together. 65536 samples of 1024 bf16 to 2 of 64 experts, streamed: scatter 73 us (403 MB),
// with weights and inner products 123 (671 MB), gather 66 (403 MB): 5.5 to 6.1 TB/s, where a large copy reaches 5.1.
constexpr int kTogether = 4;   // expert rows of a sample that are in flight together
constexpr int kLook = 16;      // expert rows that a wave looks at for empty ones

// The sample that a group of lanes works on. A whole wave's sample is uniform, and saying so puts its choices and weights
// into scalar registers and the row addresses into scalar bases.
template <bool WAVE>
__device__ __forceinline__ long long rows_sample(int lg) {
  if constexpr (WAVE) return (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  return ((long long)blockIdx.x << (8 - lg)) + (threadIdx.x >> lg);
}

// a choice's row, or -1: a plan that was tampered with does not reach past the rows
__device__ __forceinline__ long long rows_place(const RowArgs& a, int row) { return row < a.rows ? (long long)row : -1ll; }

// W: times weights; H: and inner products of the sample's row with h's
template <int DT, bool W, bool H, bool WAVE, bool NT>
__global__ __launch_bounds__(256) void rows_scatter_kernel(RowArgs a, unsigned sample_blocks) {
  typedef typename Elem<DT>::type T;
  constexpr int N = Elem<DT>::kVec;
  T* __restrict__ out = (T*)a.out;
  if (blockIdx.x >= sample_blocks) {        // rows that no sample fills are zeroed by a wave together
    const int lane = threadIdx.x & 63;
    const long long r0 = ((long long)(blockIdx.x - sample_blocks) * 4 + (threadIdx.x >> 6)) * kLook;
    const long long r = r0 + lane;
    const bool look = lane < kLook && r < a.rows;
    unsigned long long empty = __ballot(look && a.source[look ? r : 0] < 0);
    Vec<DT> zero;
    zero.w = (u32x4){0, 0, 0, 0};
    while (empty) {
      const int b = __ffsll((unsigned long long)empty) - 1;
      empty &= empty - 1;
      for (int d = lane * N; d < a.D; d += 64 * N) zero.template store<NT>(out + (r0 + b) * a.D + d, a.D - d);
    }
    return;
  }
  const int L = WAVE ? 64 : 1 << a.lg, lane = threadIdx.x & (L - 1);
  const long long t = rows_sample<WAVE>(a.lg);
  if (t >= a.T) return;
  const T* __restrict__ x = (const T*)a.x + t * a.ldx;
  const T* __restrict__ h = (const T*)a.h;
  for (int j0 = 0; j0 < a.k; j0 += kTogether) {
    long long row[kTogether];
    float w[kTogether], dot[kTogether];
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      const bool there = j0 + j < a.k;
      row[j] = there ? rows_place(a, a.position[t * a.k + j0 + j]) : -1ll;
      w[j] = W && there ? a.w[t * a.k + j0 + j] : 1.f;
      dot[j] = 0.f;
    }
    for (int d = lane * N; d < a.D; d += L * N) {
      Vec<DT> v, u[H ? kTogether : 1];
      v.template load<NT>(x + d, a.D - d);
      if constexpr (H) {
#pragma unroll
        for (int j = 0; j < kTogether; ++j)
          if (row[j] >= 0) u[j].template load<NT>(h + row[j] * a.D + d, a.D - d);
      }
#pragma unroll
      for (int j = 0; j < kTogether; ++j) {
        if (row[j] < 0) continue;
        Vec<DT> o = v;
        if constexpr (H) {
#pragma unroll
          for (int q = 0; q < N; ++q) dot[j] = fmaf(Elem<DT>::get(v.e[q]), Elem<DT>::get(u[j].e[q]), dot[j]);
        }
        if constexpr (W) {
#pragma unroll
          for (int q = 0; q < N; ++q) o.e[q] = Elem<DT>::put(Elem<DT>::get(v.e[q]) * w[j]);
        }
        o.template store<NT>(out + row[j] * a.D + d, a.D - d);
      }
    }
    if constexpr (H) {
#pragma unroll
      for (int j = 0; j < kTogether; ++j) {
        if (j0 + j >= a.k) break;
        for (int s = 1; s < L; s <<= 1) dot[j] += __shfl_xor(dot[j], s);
        if (lane == 0) a.dw[t * a.k + j0 + j] = dot[j];
      }
    }
  }
}

// P: vectors of a row in flight per lane
template <int DT, bool W, bool WAVE, int P, bool NT>
__global__ __launch_bounds__(256) void rows_gather_kernel(RowArgs a) {
  typedef typename Elem<DT>::type T;
  constexpr int N = Elem<DT>::kVec;
  const int L = WAVE ? 64 : 1 << a.lg, lane = threadIdx.x & (L - 1);
  const long long t = rows_sample<WAVE>(a.lg);
  if (t >= a.T) return;
  const T* __restrict__ h = (const T*)a.h;
  T* __restrict__ out = (T*)a.out + t * a.D;
  const int* __restrict__ position = a.position + t * a.k;
  const float* __restrict__ weight = W ? a.w + t * a.k : nullptr;
  for (int d0 = lane * N; d0 < a.D; d0 += L * N * P) {
    float sum[P][N];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int q = 0; q < N; ++q) sum[p][q] = 0.f;
    for (int j0 = 0; j0 < a.k; j0 += kTogether) {
      long long row[kTogether];
      float w[kTogether];
#pragma unroll
      for (int j = 0; j < kTogether; ++j) {
        const bool there = j0 + j < a.k;
        row[j] = there ? rows_place(a, position[j0 + j]) : -1ll;
        w[j] = W && there ? weight[j0 + j] : 1.f;
      }
      Vec<DT> v[kTogether][P];
#pragma unroll
      for (int j = 0; j < kTogether; ++j)
        if (row[j] >= 0) {
#pragma unroll
          for (int p = 0; p < P; ++p) {
            const int d = d0 + p * L * N;
            v[j][p].template load<NT>(h + row[j] * a.D + d, a.D - d);
          }
        }
#pragma unroll
      for (int j = 0; j < kTogether; ++j) {
        if (row[j] < 0) continue;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int q = 0; q < N; ++q)
            sum[p][q] = W ? fmaf(w[j], Elem<DT>::get(v[j][p].e[q]), sum[p][q]) : sum[p][q] + Elem<DT>::get(v[j][p].e[q]);
      }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int d = d0 + p * L * N;
      Vec<DT> o;
#pragma unroll
      for (int q = 0; q < N; ++q) o.e[q] = Elem<DT>::put(sum[p][q]);
      o.template store<NT>(out + d, a.D - d);
    }
  }
}

template <int DT, int L, int V>
int route_fwd_launch(const void* z, long long ldz, long long T, int E, int k, int renorm, float* w, int* ids, float* norm,
                     hipStream_t stream) {
  const long long grid = (T + 256 / L - 1) / (256 / L);
  if (grid > 0x7FFFFFFFll) return -1;
  hipLaunchKernelGGL((route_fwd_kernel<DT, L, V>), dim3((unsigned)grid), dim3(256), 0, stream,
                     (const typename Elem<DT>::type*)z, ldz, T, E, k, renorm, w, ids, norm);
  return (int)hipGetLastError();
}
template <int DT, int L, int V>
int route_bwd_launch(const void* z, long long ldz, const float* norm, const float* w, const int* ids, const float* dw,
                     long long T, int E, int k, void* dz, hipStream_t stream) {
  const long long grid = (T + 256 / L - 1) / (256 / L);
  if (grid > 0x7FFFFFFFll) return -1;
  hipLaunchKernelGGL((route_bwd_kernel<DT, L, V>), dim3((unsigned)grid), dim3(256), 0, stream,
                     (const typename Elem<DT>::type*)z, ldz, norm, w, ids, dw, T, E, k, (typename Elem<DT>::type*)dz);
  return (int)hipGetLastError();
}

// Lanes and logits per lane: the fewest lanes that hold a row in at most 16 logits each, since what crosses lanes is paid
// per row and a wave then has 64 / L rows to overlap; a lane's logits are whole 16-byte loads. A forward of more than 256
// takes 32 a lane (65536 rows, k = 8, 16 a lane and 32: 512 bf16 24 and 22 us, fp32 47 and 44; 1024 bf16 46 and 39, fp32 84 and
// 79; 256 bf16 13.7 and 13.3, not worth the registers). A backward's rows in LDS would then leave room for too few.
template <int DT>
int route_fwd_pick(const void* z, long long ldz, long long T, int E, int k, int renorm, float* w, int* ids, float* norm,
                   hipStream_t stream) {
#define RX_ROUTE(L, V) return route_fwd_launch<DT, L, V>(z, ldz, T, E, k, renorm, w, ids, norm, stream)
  if (E <= 8) RX_ROUTE(1, 8);
  if (E <= 16) RX_ROUTE(2, 8);
  if (E <= 32) RX_ROUTE(4, 8);
  if (E <= 64) RX_ROUTE(4, 16);
  if (E <= 128) RX_ROUTE(8, 16);
  if (E <= 256) RX_ROUTE(16, 16);
  if (E <= 512) RX_ROUTE(16, 32);
  RX_ROUTE(32, 32);
#undef RX_ROUTE
}
template <int DT>
int route_bwd_pick(const void* z, long long ldz, const float* norm, const float* w, const int* ids, const float* dw,
                   long long T, int E, int k, void* dz, hipStream_t stream) {
#define RX_ROUTE(L, V) return route_bwd_launch<DT, L, V>(z, ldz, norm, w, ids, dw, T, E, k, dz, stream)
  if (E <= 8) RX_ROUTE(1, 8);
  if (E <= 16) RX_ROUTE(2, 8);
  if (E <= 32) RX_ROUTE(4, 8);
  if (E <= 64) RX_ROUTE(4, 16);
  if (E <= 128) RX_ROUTE(8, 16);
  if (E <= 256) RX_ROUTE(16, 16);
  if (E <= 512) RX_ROUTE(32, 16);
  RX_ROUTE(64, 16);
#undef RX_ROUTE
}

}  // namespace

extern "C" {

unsigned long long rx_expert_layout() { return kExpertLayout; }

int rx_route_fwd(const void* z, long long ldz, int dtype, long long T, int E, int k, int renorm, float* w, int* ids,
                 float* norm, void* on) {
  hipStream_t stream = static_cast<hipStream_t>(on);
  if (T < 0 || E <= 0 || E > kMaxExperts || k <= 0 || k > kRouteMaxK || k > E) return -1;
  if (T == 0) return 0;
  if (dtype == 0) return route_fwd_pick<0>(z, ldz, T, E, k, renorm, w, ids, norm, stream);
  if (dtype == 1) return route_fwd_pick<1>(z, ldz, T, E, k, renorm, w, ids, norm, stream);
  if (dtype == 2) return route_fwd_pick<2>(z, ldz, T, E, k, renorm, w, ids, norm, stream);
  return -1;
}

int rx_route_bwd(const void* z, long long ldz, int dtype, const float* norm, const float* w, const int* ids,
                 const float* dw, long long T, int E, int k, void* dz, void* on) {
  hipStream_t stream = static_cast<hipStream_t>(on);
  if (T < 0 || E <= 0 || E > kMaxExperts || k <= 0 || k > kRouteMaxK || k > E) return -1;
  if (T == 0) return 0;
  if (dtype == 0) return route_bwd_pick<0>(z, ldz, norm, w, ids, dw, T, E, k, dz, stream);
  if (dtype == 1) return route_bwd_pick<1>(z, ldz, norm, w, ids, dw, T, E, k, dz, stream);
  if (dtype == 2) return route_bwd_pick<2>(z, ldz, norm, w, ids, dw, T, E, k, dz, stream);
  return -1;
}

int rx_expert_plan(const PlanArgs* a, int* counts, void* on) {
  hipStream_t stream = static_cast<hipStream_t>(on);
  if (a->E <= 0 || a->E > kMaxExperts || a->n < 0 || a->blocks < 1 || a->chunk <= 0 || a->chunk % kPlanThreads ||
      (long long)a->blocks * a->chunk < a->n || (a->blocks > 1 && counts == nullptr))
    return -1;
  PlanArgs p = *a;
  p.counts = a->blocks > 1 ? counts : nullptr;
  if (a->blocks > 1) {
    hipLaunchKernelGGL(plan_count_kernel, dim3((unsigned)a->blocks), dim3(kPlanThreads), 0, stream, a->ids, a->wide, a->n,
                       a->E, a->chunk, counts);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
  }
  const size_t bytes = sizeof(int) * (2 * kMaxExperts + kPlanWaves + (size_t)kPlanWaves * a->E);
  if (bytes > 65536)
    RX_CHECK(hipFuncSetAttribute((const void*)plan_rank_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  hipLaunchKernelGGL(plan_rank_kernel, dim3((unsigned)a->blocks), dim3(kPlanThreads), bytes, stream, p);
  return (int)hipGetLastError();
}

int rx_rows_scatter(const RowArgs* a, int dtype, void* on) {
  hipStream_t stream = static_cast<hipStream_t>(on);
  if (a->T < 0 || a->rows < 0 || a->k <= 0 || a->D <= 0 || a->lg < 0 || a->lg > 6 || dtype < 0 || dtype > 2) return -1;
  // (without samples only rows are zeroed)
  const bool weighted = a->T > 0 && a->w != nullptr, products = a->T > 0 && a->h != nullptr;
  if (products && (a->dw == nullptr || !weighted)) return -1;
  const long long sb = (a->T + (256 >> a->lg) - 1) >> (8 - a->lg), grid = sb + (a->rows + 4 * kLook - 1) / (4 * kLook);
  if (grid == 0) return 0;
  if (grid > 0x7FFFFFFFll) return -1;
  const dim3 g((unsigned)grid), b(256);
  const bool wave = a->lg == 6;
#define RX_SCATTER_TO(DT, W, H, WAVE, NT) \
  hipLaunchKernelGGL((rows_scatter_kernel<DT, W, H, WAVE, NT>), g, b, 0, stream, *a, (unsigned)sb)
#define RX_SCATTER_AS(DT, W, H)                                   \
  do {                                                            \
    if (wave && a->stream) RX_SCATTER_TO(DT, W, H, true, true);   \
    else if (wave) RX_SCATTER_TO(DT, W, H, true, false);          \
    else if (a->stream) RX_SCATTER_TO(DT, W, H, false, true);     \
    else RX_SCATTER_TO(DT, W, H, false, false);                   \
  } while (0)
#define RX_SCATTER(W, H)                       \
  do {                                         \
    if (dtype == 0) RX_SCATTER_AS(0, W, H);    \
    else if (dtype == 1) RX_SCATTER_AS(1, W, H); \
    else RX_SCATTER_AS(2, W, H);               \
  } while (0)
  if (products) RX_SCATTER(true, true);
  else if (weighted) RX_SCATTER(true, false);
  else RX_SCATTER(false, false);
#undef RX_SCATTER
#undef RX_SCATTER_AS
#undef RX_SCATTER_TO
  return (int)hipGetLastError();
}

int rx_rows_gather(const RowArgs* a, int dtype, void* on) {
  hipStream_t stream = static_cast<hipStream_t>(on);
  if (a->T < 0 || a->k <= 0 || a->D <= 0 || a->lg < 0 || a->lg > 6 || dtype < 0 || dtype > 2) return -1;
  const long long grid = (a->T + (256 >> a->lg) - 1) >> (8 - a->lg);
  if (grid == 0) return 0;
  if (grid > 0x7FFFFFFFll) return -1;
  const dim3 g((unsigned)grid), b(256);
  const bool wave = a->lg == 6;
#define RX_GATHER_TO(DT, W, WAVE, P, NT) hipLaunchKernelGGL((rows_gather_kernel<DT, W, WAVE, P, NT>), g, b, 0, stream, *a)
#define RX_GATHER_AS(DT, W)                                                        \
  do {                                                                             \
    if (wave && a->D > 64 * Elem<DT>::kVec) {                                      \
      if (a->stream) RX_GATHER_TO(DT, W, true, 2, true);                           \
      else RX_GATHER_TO(DT, W, true, 2, false);                                    \
    } else if (wave) {                                                             \
      if (a->stream) RX_GATHER_TO(DT, W, true, 1, true);                           \
      else RX_GATHER_TO(DT, W, true, 1, false);                                    \
    } else {                                                                       \
      if (a->stream) RX_GATHER_TO(DT, W, false, 1, true);                          \
      else RX_GATHER_TO(DT, W, false, 1, false);                                   \
    }                                                                              \
  } while (0)
#define RX_GATHER(W)                       \
  do {                                     \
    if (dtype == 0) RX_GATHER_AS(0, W);    \
    else if (dtype == 1) RX_GATHER_AS(1, W); \
    else RX_GATHER_AS(2, W);               \
  } while (0)
  if (a->w != nullptr) RX_GATHER(true);
  else RX_GATHER(false);
#undef RX_GATHER
#undef RX_GATHER_AS
#undef RX_GATHER_TO
  return (int)hipGetLastError();
}

}  // extern "C"
