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
// scatter and gather are each other's gradients; every kernel works sample by sample, so that x, dy and y cross memory
// once, the sums of a sample are one lane group's in a fixed order, and nothing needs atomics on floats.
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
  // n: elements there (a row's last vector may be short)
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= Elem<DT>::kVec) {
      w = *(const u32x4_u*)p;
    } else {
      w = (u32x4){0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < Elem<DT>::kVec - 1; ++i)
        if (i < n) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p, int n) const {
    if (n >= Elem<DT>::kVec) {
      *(u32x4_u*)p = w;
    } else {
#pragma unroll
      for (int i = 0; i < Elem<DT>::kVec - 1; ++i)
        if (i < n) p[i] = e[i];
    }
  }
};

// ------------------------------------------------------------------------------------------------ router
constexpr int kRouteMaxK = 32;

// L lanes hold a row, V logits each: element i * L + lane
template <int DT, int L, int V>
__global__ __launch_bounds__(256) void route_fwd_kernel(const typename Elem<DT>::type* __restrict__ z, long long ldz,
                                                        long long T, int E, int k, int renorm, float* __restrict__ w,
                                                        int* __restrict__ ids, float* __restrict__ norm) {
  const int lane = threadIdx.x % L;
  const long long t = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (t >= T) return;
  const float kNone = -__builtin_huge_valf();
  float v[V];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * L + lane;
    v[i] = e < E ? Elem<DT>::get(z[t * ldz + e]) : kNone;
    bad |= v[i] != v[i];
  }
  constexpr int kSlots = (kRouteMaxK + L - 1) / L;
  float zs[kSlots];
  int is[kSlots];
  float peak = 0.f, total = 0.f;
  for (int j = 0; j < k; ++j) {
    float best = kNone;
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (v[i] > best) {
        best = v[i];
        at = i * L + lane;
      }
#pragma unroll
    for (int d = 1; d < L; d <<= 1) {
      const float ob = __shfl_xor(best, d);
      const int oa = __shfl_xor(at, d);
      const bool take = ob > best || (ob == best && oa < at);
      best = take ? ob : best;
      at = take ? oa : at;
    }
    if (j == 0) {
      peak = best > kNone ? best : 0.f;
      if (!renorm) {
#pragma unroll
        for (int i = 0; i < V; ++i) total += expf(v[i] - peak);
#pragma unroll
        for (int d = 1; d < L; d <<= 1) total += __shfl_xor(total, d);
      }
    }
    const float ex = best > kNone ? expf(best - peak) : 0.f;
    if (renorm) total += ex;
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
      if (j == s * L + lane) {
        zs[s] = ex;
        is[s] = best > kNone ? at : -1;
      }
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (at == i * L + lane) v[i] = kNone;
  }
  // a NaN in the row shows in all of its weights
  const unsigned long long rows = __ballot(bad);
  const int shift = (threadIdx.x & 63) / L * L;
  const bool any = ((rows >> shift) & (L == 64 ? ~0ull : (1ull << (L & 63)) - 1)) != 0;
  const float inv = any ? __uint_as_float(0x7FC00000u) : total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    const int j = s * L + lane;
    if (j < k) {
      w[t * k + j] = zs[s] * inv;
      ids[t * k + j] = is[s];
    }
  }
  if (norm != nullptr && lane == 0) {
    norm[2 * t] = peak;
    norm[2 * t + 1] = inv;
  }
}

template <int DT, int L, int V>
__global__ __launch_bounds__(256) void route_bwd_kernel(const typename Elem<DT>::type* __restrict__ z, long long ldz,
                                                        const float* __restrict__ norm, const float* __restrict__ w,
                                                        const int* __restrict__ ids, const float* __restrict__ dw,
                                                        long long T, int E, int k,
                                                        typename Elem<DT>::type* __restrict__ dz) {
  const int lane = threadIdx.x % L;
  const long long t = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (t >= T) return;
  float s = 0.f;
  for (int j = 0; j < k; ++j) s = ids[t * k + j] >= 0 ? fmaf(w[t * k + j], dw[t * k + j], s) : s;
  float g[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * L + lane;
    g[i] = 0.f;
    if (norm != nullptr && e < E)
      g[i] = -s * (expf(Elem<DT>::get(z[t * ldz + e]) - norm[2 * t]) * norm[2 * t + 1]);
  }
  for (int j = 0; j < k; ++j) {
    const int e = ids[t * k + j];
    if (e < 0) continue;
    const float add = w[t * k + j] * (norm != nullptr ? dw[t * k + j] : dw[t * k + j] - s);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (e == i * L + lane) g[i] += add;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * L + lane;
    if (e < E) dz[t * E + e] = Elem<DT>::put(g[i]);
  }
}

// ------------------------------------------------------------------------------------------------ plan
constexpr int kPlanWaves = 16, kPlanThreads = 64 * kPlanWaves;
constexpr int kMaxExperts = 1024;

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

struct PlanArgs {
  const void* ids;
  int wide, n, E, chunk, blocks, capacity, rows, pad_;
  const int* counts;    // [blocks][E] (null with one block)
  int* position;        // [n]
  int* source;          // [rows]
  int* load;            // [E]
  int* offsets;         // [E + 1]
};

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
      for (int r = before[e] + tid; r < a.capacity; r += kPlanThreads) a.source[e * a.capacity + r] = -1;
  } else {
    for (int r = all + blockIdx.x * kPlanThreads + tid; r < a.rows; r += gridDim.x * kPlanThreads) a.source[r] = -1;
  }
  int bits = 0;
  while ((1 << bits) < E) ++bits;
  volatile int* mynext = next + wave * E;
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
    __builtin_amdgcn_wave_barrier();
    if (e >= 0 && (same >> lane) == 1ull) mynext[e] = rank + 1;     // the last of its lanes
    __builtin_amdgcn_wave_barrier();
    if (there) {
      a.position[i] = row;
      if (row >= 0) a.source[row] = (int)i;
    }
  }
}

// ------------------------------------------------------------------------------------------------ rows
struct RowArgs {
  long long T, rows, ldx;     // samples, expert rows, elements between samples' rows (x)
  int k, D, lg, pad_;         // lg: log2 of the lanes that work on a sample
  const int* position;        // [T][k]
  const int* source;          // [rows]
  const void* x;              // scatter: samples' rows in; gather: not used
  const float* w;             // [T][k] or null
  const void* h;              // scatter: expert rows to take products with, or null; gather: expert rows in
  void* out;                  // scatter: expert rows out; gather: samples' rows out
  float* dw;                  // scatter with h: [T][k]
};

template <int DT>
__global__ __launch_bounds__(256) void rows_scatter_kernel(RowArgs a, unsigned sample_blocks) {
  typedef typename Elem<DT>::type T;
  constexpr int N = Elem<DT>::kVec;
  T* out = (T*)a.out;
  if (blockIdx.x >= sample_blocks) {        // rows that no sample fills: 64 looked at by each wave, zeroed together
    const int lane = threadIdx.x & 63;
    const long long r0 = ((long long)(blockIdx.x - sample_blocks) * 4 + (threadIdx.x >> 6)) * 64;
    const long long r = r0 + lane;
    unsigned long long empty = __ballot(r < a.rows && a.source[r < a.rows ? r : 0] < 0);
    Vec<DT> zero;
    zero.w = (u32x4){0, 0, 0, 0};
    while (empty) {
      const int b = __ffsll((unsigned long long)empty) - 1;
      empty &= empty - 1;
      for (int d = lane * N; d < a.D; d += 64 * N) zero.store(out + (r0 + b) * a.D + d, a.D - d);
    }
    return;
  }
  const int L = 1 << a.lg, lane = threadIdx.x & (L - 1);
  const long long t = ((long long)blockIdx.x << (8 - a.lg)) + (threadIdx.x >> a.lg);
  if (t >= a.T) return;
  const T* x = (const T*)a.x + t * a.ldx;
  const T* h = (const T*)a.h;
  for (int j = 0; j < a.k; ++j) {
    const long long row = a.position[t * a.k + j];
    float dot = 0.f;
    if (row >= 0) {
      const float w = a.w != nullptr ? a.w[t * a.k + j] : 1.f;
      for (int d = lane * N; d < a.D; d += L * N) {
        Vec<DT> v;
        v.load(x + d, a.D - d);
        if (h != nullptr) {
          Vec<DT> u;
          u.load(h + row * a.D + d, a.D - d);
#pragma unroll
          for (int q = 0; q < N; ++q) dot = fmaf(Elem<DT>::get(v.e[q]), Elem<DT>::get(u.e[q]), dot);
        }
        if (a.w != nullptr) {
#pragma unroll
          for (int q = 0; q < N; ++q) v.e[q] = Elem<DT>::put(Elem<DT>::get(v.e[q]) * w);
        }
        v.store(out + row * a.D + d, a.D - d);
      }
    }
    if (a.dw != nullptr) {
      for (int s = 1; s < L; s <<= 1) dot += __shfl_xor(dot, s);
      if (lane == 0) a.dw[t * a.k + j] = dot;
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void rows_gather_kernel(RowArgs a) {
  typedef typename Elem<DT>::type T;
  constexpr int N = Elem<DT>::kVec;
  const int L = 1 << a.lg, lane = threadIdx.x & (L - 1);
  const long long t = ((long long)blockIdx.x << (8 - a.lg)) + (threadIdx.x >> a.lg);
  if (t >= a.T) return;
  const T* h = (const T*)a.h;
  T* out = (T*)a.out + t * a.D;
  for (int d = lane * N; d < a.D; d += L * N) {
    float sum[N];
#pragma unroll
    for (int q = 0; q < N; ++q) sum[q] = 0.f;
    for (int j = 0; j < a.k; ++j) {
      const long long row = a.position[t * a.k + j];
      if (row < 0) continue;
      const float w = a.w != nullptr ? a.w[t * a.k + j] : 1.f;
      Vec<DT> v;
      v.load(h + row * a.D + d, a.D - d);
#pragma unroll
      for (int q = 0; q < N; ++q) sum[q] = fmaf(w, Elem<DT>::get(v.e[q]), sum[q]);
    }
    Vec<DT> o;
#pragma unroll
    for (int q = 0; q < N; ++q) o.e[q] = Elem<DT>::put(sum[q]);
    o.store(out + d, a.D - d);
  }
}

template <int DT, int L, int V>
int route_launch(int bwd, const void* z, long long ldz, const float* norm, float* w, int* ids, const float* dw,
                 long long T, int E, int k, int renorm, float* norm_out, void* dz, hipStream_t stream) {
  typedef typename Elem<DT>::type S;
  const long long grid = (T + 256 / L - 1) / (256 / L);
  if (grid > 0x7FFFFFFFll) return -1;
  if (bwd)
    hipLaunchKernelGGL((route_bwd_kernel<DT, L, V>), dim3((unsigned)grid), dim3(256), 0, stream, (const S*)z, ldz, norm,
                       w, ids, dw, T, E, k, (S*)dz);
  else
    hipLaunchKernelGGL((route_fwd_kernel<DT, L, V>), dim3((unsigned)grid), dim3(256), 0, stream, (const S*)z, ldz, T, E,
                       k, renorm, w, ids, norm_out);
  return (int)hipGetLastError();
}

template <int DT>
int route_pick(int bwd, const void* z, long long ldz, const float* norm, float* w, int* ids, const float* dw, long long T,
               int E, int k, int renorm, float* norm_out, void* dz, hipStream_t stream) {
#define RX_ROUTE(L, V) \
  return route_launch<DT, L, V>(bwd, z, ldz, norm, w, ids, dw, T, E, k, renorm, norm_out, dz, stream)
  if (E <= 16) RX_ROUTE(4, 4);
  if (E <= 64) RX_ROUTE(8, 8);
  if (E <= 128) RX_ROUTE(16, 8);
  if (E <= 256) RX_ROUTE(16, 16);
  if (E <= 512) RX_ROUTE(32, 16);
  RX_ROUTE(64, 16);
#undef RX_ROUTE
}

}  // namespace

extern "C" {

void rx_expert_sizes(int* out) {   // mirrored by raydp_amd/ops/expert_ops.py
  out[0] = (int)sizeof(PlanArgs);
  out[1] = (int)sizeof(RowArgs);
  out[2] = kMaxExperts;
  out[3] = kRouteMaxK;
}

// dtype: 0 fp32, 1 bf16, 2 fp16. norm: [T][2] peak and 1 / sum, written when not null
int rx_route_fwd(const void* z, long long ldz, int dtype, long long T, int E, int k, int renorm, float* w, int* ids,
                 float* norm, hipStream_t stream) {
  if (T < 0 || E <= 0 || E > kMaxExperts || k <= 0 || k > kRouteMaxK || k > E) return -1;
  if (T == 0) return 0;
  if (dtype == 0) return route_pick<0>(0, z, ldz, nullptr, w, ids, nullptr, T, E, k, renorm, norm, nullptr, stream);
  if (dtype == 1) return route_pick<1>(0, z, ldz, nullptr, w, ids, nullptr, T, E, k, renorm, norm, nullptr, stream);
  if (dtype == 2) return route_pick<2>(0, z, ldz, nullptr, w, ids, nullptr, T, E, k, renorm, norm, nullptr, stream);
  return -1;
}

// norm null: softmax over the chosen ones (z is not read)
int rx_route_bwd(const void* z, long long ldz, int dtype, const float* norm, const float* w, const int* ids,
                 const float* dw, long long T, int E, int k, void* dz, hipStream_t stream) {
  if (T < 0 || E <= 0 || E > kMaxExperts || k <= 0 || k > kRouteMaxK || k > E) return -1;
  if (T == 0) return 0;
  float* wm = const_cast<float*>(w);
  int* im = const_cast<int*>(ids);
  if (dtype == 0) return route_pick<0>(1, z, ldz, norm, wm, im, dw, T, E, k, 0, nullptr, dz, stream);
  if (dtype == 1) return route_pick<1>(1, z, ldz, norm, wm, im, dw, T, E, k, 0, nullptr, dz, stream);
  if (dtype == 2) return route_pick<2>(1, z, ldz, norm, wm, im, dw, T, E, k, 0, nullptr, dz, stream);
  return -1;
}

// counts: blocks * E ints of scratch (not read or written with one block)
int rx_expert_plan(const PlanArgs* a, int* counts, hipStream_t stream) {
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

int rx_rows_scatter(const RowArgs* a, int dtype, hipStream_t stream) {
  if (a->T < 0 || a->rows < 0 || a->k <= 0 || a->D <= 0 || a->lg < 0 || a->lg > 6 || dtype < 0 || dtype > 2) return -1;
  const long long sb = (a->T + (256 >> a->lg) - 1) >> (8 - a->lg), grid = sb + (a->rows + 255) / 256;
  if (grid == 0) return 0;
  if (grid > 0x7FFFFFFFll) return -1;
  const dim3 g((unsigned)grid), b(256);
  if (dtype == 0) hipLaunchKernelGGL((rows_scatter_kernel<0>), g, b, 0, stream, *a, (unsigned)sb);
  else if (dtype == 1) hipLaunchKernelGGL((rows_scatter_kernel<1>), g, b, 0, stream, *a, (unsigned)sb);
  else hipLaunchKernelGGL((rows_scatter_kernel<2>), g, b, 0, stream, *a, (unsigned)sb);
  return (int)hipGetLastError();
}

int rx_rows_gather(const RowArgs* a, int dtype, hipStream_t stream) {
  if (a->T < 0 || a->k <= 0 || a->D <= 0 || a->lg < 0 || a->lg > 6 || dtype < 0 || dtype > 2) return -1;
  const long long grid = (a->T + (256 >> a->lg) - 1) >> (8 - a->lg);
  if (grid == 0) return 0;
  if (grid > 0x7FFFFFFFll) return -1;
  const dim3 g((unsigned)grid), b(256);
  if (dtype == 0) hipLaunchKernelGGL((rows_gather_kernel<0>), g, b, 0, stream, *a);
  else if (dtype == 1) hipLaunchKernelGGL((rows_gather_kernel<1>), g, b, 0, stream, *a);
  else hipLaunchKernelGGL((rows_gather_kernel<2>), g, b, 0, stream, *a);
  return (int)hipGetLastError();
}

}  // extern "C"
