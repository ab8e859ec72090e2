// AdamW over many tensors with the moments in 8 or 32 bits, the global gradient norm that clips it, and the scaling of
// gradients by that norm (raydp_amd/ops/fused_optim.py FusedAdamW, clip_grad_norm_, decode_moments).
//
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2          g taken times the clip factor
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A step is up to three kinds of launches on one stream: norm_part_kernel (only with clipping), aw_prep_kernel (one
// workgroup: finishes the norm, advances the tensors' step words, works out what one step has in common per tensor) and
// aw_step_kernel (everything elementwise). Nothing of a step lives on the host, so a captured step replays correctly.
//
// Moments in 8 bits. 256 consecutive elements of a tensor share a power-of-two scale 2^e per moment, one byte each. m is
// sign + 4 exponent + 3 mantissa bits, v (never negative) 5 exponent + 3 mantissa bits, both with gradual underflow. v
// gets the longer exponent because its square root divides: both reach 2^-16 of their block's largest magnitude. After
// scaling by a power of two (ldexp, exact) such a code IS the top of an fp32 bit pattern, so coding is an integer add and
// a shift. The add is a dither: rounding to nearest would never move v, whose change per step (1 - b2 = 0.1 %) is far
// below half a code's spacing (6 %); with the dither the expectation of the stored value is the value.
// e is the exponent of the block's maximum once that is rounded up to 3 mantissa bits, so no rounding overflows. A byte
// of 255 marks a block whose values are not finite: it decodes to NaN, as fp32 moments would show it.
// m and v are computed as separately rounded products and sums: any IEEE fp32 implementation gets the same codes.
#include "rx_common.h"

namespace {

constexpr int kAwMax = 48;      // tensors in one step launch (kernel arguments under 4 KiB)
constexpr int kPrepMax = 256;   // tensors in one preparation launch (one thread each)
constexpr int kNormMax = 128;   // tensors in one norm / scale launch
constexpr int kBlk = 256;       // elements that share a scale: 4 per lane of one wave

// dither: 2^32 / golden ratio and the fractional bits of sqrt(2), sqrt(3) as odd multipliers
constexpr uint32_t kPhi = 0x9E3779B1u, kSq2 = 0x6A09E667u, kSq3 = 0xBB67AE85u;

__device__ __forceinline__ uint32_t aw_mix(uint32_t x) {
  x = (x ^ (x >> 16)) * kSq2;
  x = (x ^ (x >> 15)) * kSq3;
  return x ^ (x >> 16);
}

struct AwHead {      // one per launch group of a step
  float gscale;      // what gradients are multiplied with (clip factor, -1 to maximize)
  int skip;          // 1: the norm is not finite, the step is left out
};

struct AwTensor {    // what one step has in common for a tensor
  float nlr_bc1;     // -lr / (1 - b1^t)
  float decay;       // 1 - lr wd
  float rs_bc2;      // 1 / sqrt(1 - b2^t)
  uint32_t key;      // of its dither in this step
};

struct AwPrep {
  int n, maximize, npart, first;   // first: index of this launch's first tensor in tensors[]
  double lr, wd, b1, b2, max_norm; // max_norm < 0: no clipping
  const float* lr_dev;             // not null: the learning rate, on the device
  const double* part;              // npart partial sums of squared gradients
  AwHead* head;
  AwTensor* tensors;
  float* norm;                     // not null: where the norm goes
  uint32_t seed, pad_;
  float* step[kPrepMax];           // the tensors' step words
  int ordinal[kPrepMax];           // their places in the optimizer
};

struct AwStep {
  int n, pad_;
  float b1, omb1, b2, omb2, eps, pad2_;
  const AwHead* head;
  const AwTensor* tensors;         // of this launch's first tensor
  void* p[kAwMax];
  const void* g[kAwMax];
  void* m[kAwMax];
  void* v[kAwMax];
  uint8_t* sc[kAwMax];             // [blocks][2] scale bytes (8-bit moments)
  u16* img[kAwMax];                // bf16 image of an fp32 p (null: none)
  long long len[kAwMax];
  unsigned start[kAwMax + 1];      // first chunk of each tensor
};

struct NormArgs {
  int n, bf16_mask_;
  double* part;                    // one partial sum per workgroup
  unsigned chunks, pad_;
  const void* g[kNormMax];
  long long len[kNormMax];
  unsigned start[kNormMax + 1];
  unsigned char bf16[kNormMax];
};

struct ScaleArgs {
  NormArgs t;                      // t.part: the partial sums to finish
  int npart, pad_;
  double max_norm;
  float* norm;
};

// the tensor that a chunk belongs to: start[] is ascending, wave-uniform
template <class A>
__device__ __forceinline__ int aw_find(const A& a, int n, unsigned c) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.start[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint32_t aw_wavemax(uint32_t v) {
  v = max(v, rx_dppu<RX_DPP_XOR1>(v));
  v = max(v, rx_dppu<RX_DPP_XOR2>(v));
  v = max(v, rx_dppu<RX_DPP_HALF_MIRROR>(v));
  v = max(v, rx_dppu<RX_DPP_MIRROR>(v));
  const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(p[0], p[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(q[0], q[1]);
}

// biased scale exponent of a block from the largest magnitude's bits (NaN and infinity: 255)
__device__ __forceinline__ int aw_scale(uint32_t top) { return (int)((top + 0xFFFFFu) >> 23); }
__device__ __forceinline__ int aw_exp(int s) { return (s > 0 ? s : 1) - 127; }

// code <-> value: a value scaled so that the code's smallest normal lands on fp32's is a code in its top bits
constexpr int kMShift = 112, kVShift = 96;   // 126 - 14, 126 - 30
__device__ __forceinline__ float aw_dec_m(uint32_t c, int e) {
  const float a = ldexpf(__uint_as_float((c & 0x7Fu) << 20), e + kMShift);
  return (c & 0x80u) ? -a : a;
}
__device__ __forceinline__ float aw_dec_v(uint32_t c, int e) {
  return ldexpf(__uint_as_float(c << 20), e + kVShift);
}
__device__ __forceinline__ uint32_t aw_enc_m(float m, int e, uint32_t rnd16) {
  const uint32_t a = __float_as_uint(ldexpf(fabsf(m), -e - kMShift));
  return ((a + (rnd16 * 16u + 8u)) >> 20) | ((__float_as_uint(m) >> 31) << 7);
}
__device__ __forceinline__ uint32_t aw_enc_v(float v, int e, uint32_t rnd16) {
  const uint32_t a = __float_as_uint(ldexpf(v, -e - kVShift));
  const uint32_t c = (a + (rnd16 * 16u + 8u)) >> 20;
  return (v > 0.f && c == 0u) ? 1u : c;      // what is not zero stays so: it is divided by
}

__device__ __forceinline__ u16 aw_dither_bf16(float x, uint32_t rnd16) {
  const uint32_t b = __float_as_uint(x);
  return (u16)(((b & 0x7FFFFFFFu) > 0x7F800000u ? b : b + rnd16) >> 16);
}

// 4 consecutive elements from i on; n: how many there are (<= 4)
template <bool BF16>
__device__ __forceinline__ f32x4 aw_load4(const void* base, long long i, int n, bool vec) {
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if constexpr (BF16) {
    const u16* s = (const u16*)base + i;
    if (vec && n == 4) {
      const uint2 w = *(const uint2*)s;
      r[0] = rx_bf2f((u16)w.x);
      r[1] = __uint_as_float(w.x & 0xFFFF0000u);
      r[2] = rx_bf2f((u16)w.y);
      r[3] = __uint_as_float(w.y & 0xFFFF0000u);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < n) r[k] = rx_bf2f(s[k]);
    }
  } else {
    const float* s = (const float*)base + i;
    if (vec && n == 4) {
      r = *(const f32x4*)s;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < n) r[k] = s[k];
    }
  }
  return r;
}

__device__ __forceinline__ void aw_store4(float* s, const f32x4& r, int n, bool vec) {
  if (vec && n == 4) {
    *(f32x4*)s = r;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) s[k] = r[k];
  }
}
__device__ __forceinline__ void aw_store4h(u16* s, const u16* r, int n, bool vec) {
  if (vec && n == 4) {
    *(uint2*)s = make_uint2(r[0] | (uint32_t)r[1] << 16, r[2] | (uint32_t)r[3] << 16);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) s[k] = r[k];
  }
}
__device__ __forceinline__ uint32_t aw_load4c(const uint8_t* s, int n) {
  if (n == 4) return *(const uint32_t*)s;
  uint32_t r = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < n) r |= (uint32_t)s[k] << (8 * k);
  return r;
}
__device__ __forceinline__ void aw_store4c(uint8_t* s, uint32_t c, int n) {
  if (n == 4) {
    *(uint32_t*)s = c;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) s[k] = (uint8_t)(c >> (8 * k));
  }
}

constexpr int kStepUnroll = 1;                        // scale blocks per wave
constexpr int kStepChunk = 4 * kBlk * kStepUnroll;    // elements per workgroup of 4 waves

template <bool BITS8, bool BF16>
__global__ __launch_bounds__(256) void aw_step_kernel(AwStep a) {
  const AwHead head = *a.head;
  if (head.skip) return;
  const int t = aw_find(a, a.n, blockIdx.x);
  const AwTensor k = a.tensors[t];
  const long long n = a.len[t];
  void* p = a.p[t];
  const void* g = a.g[t];
  u16* img = BF16 ? nullptr : a.img[t];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool vec = (((uintptr_t)p | (uintptr_t)g | (uintptr_t)img * 2) & 15) == 0;
#pragma unroll
  for (int u = 0; u < kStepUnroll; ++u) {
    const long long blk = (long long)(blockIdx.x - a.start[t]) * (4 * kStepUnroll) + wave * kStepUnroll + u;
    const long long i = blk * kBlk + lane * 4;
    const int left = n - i >= 4 ? 4 : n - i > 0 ? (int)(n - i) : 0;
    if (blk * kBlk >= n) break;                       // (wave-uniform)
    f32x4 pv = aw_load4<BF16>(p, i, left, vec), gv = aw_load4<BF16>(g, i, left, vec);
    f32x4 mv, vv;
    uint8_t* sc = nullptr;
    if constexpr (BITS8) {
      sc = a.sc[t] + blk * 2;
      const int sm = sc[0], sv = sc[1];
      const uint32_t mc = aw_load4c((const uint8_t*)a.m[t] + i, left), vc = aw_load4c((const uint8_t*)a.v[t] + i, left);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        mv[q] = aw_dec_m((mc >> (8 * q)) & 0xFFu, aw_exp(sm));
        vv[q] = aw_dec_v((vc >> (8 * q)) & 0xFFu, aw_exp(sv));
      }
      if (sm == 255 || sv == 255) {
        const float nan = __uint_as_float(0x7FC00000u);
        mv = sm == 255 ? (f32x4){nan, nan, nan, nan} : mv;
        vv = sv == 255 ? (f32x4){nan, nan, nan, nan} : vv;
      }
    } else {
      mv = aw_load4<false>(a.m[t], i, left, true);
      vv = aw_load4<false>(a.v[t], i, left, true);
    }
    uint32_t h[4];
    uint32_t mtop = 0, vtop = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      {
#pragma clang fp contract(off)
        const float gq = gv[q] * head.gscale;
        mv[q] = a.b1 * mv[q] + a.omb1 * gq;
        vv[q] = a.b2 * vv[q] + a.omb2 * (gq * gq);
      }
      // square root and quotient to 1 ulp each: the update is about 1e-3 of p
      const float den = fmaf(__builtin_amdgcn_sqrtf(vv[q]), k.rs_bc2, a.eps);
      pv[q] = fmaf(k.nlr_bc1, mv[q] * __builtin_amdgcn_rcpf(den), pv[q] * k.decay);
      if (q < left) {
        mtop = max(mtop, __float_as_uint(mv[q]) & 0x7FFFFFFFu);
        vtop = max(vtop, __float_as_uint(vv[q]) & 0x7FFFFFFFu);
      }
      if constexpr (BITS8 || BF16) {
        const unsigned long long j = (unsigned long long)i + q;
        h[q] = aw_mix((uint32_t)j * kPhi + (uint32_t)(j >> 32) * kSq2 + k.key);
      }
    }
    if constexpr (BITS8) {
      const int sm = aw_scale(aw_wavemax(mtop)), sv = aw_scale(aw_wavemax(vtop));
      uint32_t mc = 0, vc = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        mc |= aw_enc_m(mv[q], aw_exp(sm), h[q] & 0xFFFFu) << (8 * q);
        vc |= aw_enc_v(vv[q], aw_exp(sv), h[q] >> 16) << (8 * q);
      }
      if (sm == 255) mc = 0;
      if (sv == 255) vc = 0;
      aw_store4c((uint8_t*)a.m[t] + i, mc, left);
      aw_store4c((uint8_t*)a.v[t] + i, vc, left);
      if (lane == 0) {
        sc[0] = (uint8_t)sm;
        sc[1] = (uint8_t)sv;
      }
    } else {
      aw_store4((float*)a.m[t] + i, mv, left, true);
      aw_store4((float*)a.v[t] + i, vv, left, true);
    }
    if constexpr (BF16) {
      // no master copy: rounded with the dither, so that updates under half a step of p are not lost
      u16 o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = aw_dither_bf16(pv[q], (h[q] * kSq2) >> 16);
      aw_store4h((u16*)p + i, o, left, vec);
    } else {
      aw_store4((float*)p + i, pv, left, vec);
      if (img != nullptr) {
        u16 o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = rx_f2bf(pv[q]);
        aw_store4h(img + i, o, left, vec);
      }
    }
  }
}

// sum over a workgroup of 256 in a fixed order; the result is valid in thread 0
__device__ __forceinline__ double aw_blocksum(double s, double* lds) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

__device__ __forceinline__ double aw_partsum(const double* part, int npart, double* lds) {
  double s = 0.0;
  for (int i = threadIdx.x; i < npart; i += 256) s += part[i];
  return aw_blocksum(s, lds);
}

// min(1, max / (norm + 1e-6)): the factor of torch.nn.utils.clip_grad_norm_
__device__ __forceinline__ float aw_clip(double norm, double max_norm) {
  const double c = max_norm / (norm + 1e-6);
  return (float)(c < 1.0 ? c : c >= 1.0 ? 1.0 : c);   // (a NaN stays one)
}

__global__ __launch_bounds__(256) void aw_prep_kernel(AwPrep a) {
  __shared__ double lds[4];
  float scale = 1.f;
  int skip = 0;
  if (a.max_norm >= 0.0) {
    const double norm = sqrt(aw_partsum(a.part, a.npart, lds));
    scale = aw_clip(norm, a.max_norm);
    skip = !(norm < __builtin_huge_val());
    if (threadIdx.x == 0 && a.norm != nullptr) *a.norm = (float)norm;
  }
  if (threadIdx.x == 0) {
    a.head->gscale = a.maximize ? -scale : scale;
    a.head->skip = skip;
  }
  const int i = threadIdx.x;
  if (i >= a.n || skip) return;
  const float step = *a.step[i] + 1.f;
  *a.step[i] = step;
  const double t = (double)step, lr = a.lr_dev != nullptr ? (double)*a.lr_dev : a.lr;
  AwTensor k;
  k.nlr_bc1 = (float)(-lr / (1.0 - pow(a.b1, t)));
  k.decay = (float)(1.0 - lr * a.wd);
  k.rs_bc2 = (float)(1.0 / sqrt(1.0 - pow(a.b2, t)));
  k.key = aw_mix(aw_mix(a.seed + (uint32_t)a.ordinal[i] * kPhi) + (uint32_t)step);
  a.tensors[a.first + i] = k;
}

// Sums of squares in 64 bits: the norm then does not depend on the order of the sum in any of its 32 bits but by chance.
constexpr int kNormChunk = 4096;

template <bool BF16>
__device__ __forceinline__ double aw_squares(const void* g, long long i, long long n, bool vec) {
  double s = 0.0;
#pragma unroll
  for (int u = 0; u < kNormChunk / 1024; ++u) {
    const long long j = i + u * 1024 + threadIdx.x * 4;
    const int left = n - j >= 4 ? 4 : n - j > 0 ? (int)(n - j) : 0;
    const f32x4 v = aw_load4<BF16>(g, j, left, vec);
#pragma unroll
    for (int q = 0; q < 4; ++q) s = fma((double)v[q], (double)v[q], s);
  }
  return s;
}

__global__ __launch_bounds__(256) void norm_part_kernel(NormArgs a) {
  __shared__ double lds[4];
  double s = 0.0;
  for (unsigned c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const int t = aw_find(a, a.n, c);
    const void* g = a.g[t];
    const long long i = (long long)(c - a.start[t]) * kNormChunk;
    const bool vec = ((uintptr_t)g & 15) == 0;
    s += a.bf16[t] ? aw_squares<true>(g, i, a.len[t], vec) : aw_squares<false>(g, i, a.len[t], vec);
  }
  s = aw_blocksum(s, lds);
  if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

// g *= min(1, max_norm / (norm + 1e-6)); every workgroup finishes the norm itself (a few KB out of L2), which saves a
// launch between the two passes; with a factor of 1 nothing is touched
__global__ __launch_bounds__(256) void norm_scale_kernel(ScaleArgs a) {
  __shared__ double lds[4];
  const double norm = sqrt(aw_partsum(a.t.part, a.npart, lds));
  const float f = aw_clip(norm, a.max_norm);
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.norm != nullptr) *a.norm = (float)norm;
  if (f == 1.f) return;
  for (unsigned c = blockIdx.x; c < a.t.chunks; c += gridDim.x) {
    const int t = aw_find(a.t, a.t.n, c);
    void* g = const_cast<void*>(a.t.g[t]);
    const long long n = a.t.len[t];
    const bool vec = ((uintptr_t)g & 15) == 0;
#pragma unroll
    for (int u = 0; u < kNormChunk / 1024; ++u) {
      const long long j = (long long)(c - a.t.start[t]) * kNormChunk + u * 1024 + threadIdx.x * 4;
      const int left = n - j >= 4 ? 4 : n - j > 0 ? (int)(n - j) : 0;
      if (left <= 0) continue;
      if (a.t.bf16[t]) {
        const f32x4 v = aw_load4<true>(g, j, left, vec);
        u16 o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = rx_f2bf(v[q] * f);
        aw_store4h((u16*)g + j, o, left, vec);
      } else {
        f32x4 v = aw_load4<false>(g, j, left, vec);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] *= f;
        aw_store4((float*)g + j, v, left, vec);
      }
    }
  }
}

// codes -> the values they stand for (at most 4 significant bits: exact in bf16 too)
template <bool BF16>
__global__ __launch_bounds__(256) void aw_decode_kernel(const uint8_t* m, const uint8_t* v, const uint8_t* sc, void* mo,
                                                        void* vo, long long n) {
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (long long)gridDim.x * 1024) {
    const int left = n - i >= 4 ? 4 : (int)(n - i);
    const int sm = sc[(i / kBlk) * 2], sv = sc[(i / kBlk) * 2 + 1];
    const uint32_t mc = aw_load4c(m + i, left), vc = aw_load4c(v + i, left);
    const float nan = __uint_as_float(0x7FC00000u);
    f32x4 mv, vv;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      mv[q] = sm == 255 ? nan : aw_dec_m((mc >> (8 * q)) & 0xFFu, aw_exp(sm));
      vv[q] = sv == 255 ? nan : aw_dec_v((vc >> (8 * q)) & 0xFFu, aw_exp(sv));
    }
    if constexpr (BF16) {
      u16 a[4], b[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        a[q] = rx_f2bf(mv[q]);
        b[q] = rx_f2bf(vv[q]);
      }
      aw_store4h((u16*)mo + i, a, left, true);
      aw_store4h((u16*)vo + i, b, left, true);
    } else {
      aw_store4((float*)mo + i, mv, left, true);
      aw_store4((float*)vo + i, vv, left, true);
    }
  }
}

}  // namespace

extern "C" {

void rx_aw_sizes(int* out) {   // struct sizes and limits that raydp_amd/ops/fused_optim.py mirrors
  out[0] = (int)sizeof(AwPrep);
  out[1] = (int)sizeof(AwStep);
  out[2] = (int)sizeof(NormArgs);
  out[3] = (int)sizeof(ScaleArgs);
  out[4] = kAwMax;
  out[5] = kPrepMax;
  out[6] = kNormMax;
  out[7] = kStepChunk;
  out[8] = kNormChunk;
}

int rx_aw_prep(const AwPrep* a, hipStream_t stream) {
  if (a->n < 0 || a->n > kPrepMax) return -1;
  hipLaunchKernelGGL(aw_prep_kernel, dim3(1), dim3(256), 0, stream, *a);
  return (int)hipGetLastError();
}

int rx_aw_step(const AwStep* a, int bits, int bf16, hipStream_t stream) {
  if (a->n <= 0 || a->n > kAwMax || (bits != 8 && bits != 32)) return -1;
  const unsigned grid = a->start[a->n];
  if (grid == 0) return 0;
  if (grid > 0x7FFFFFFFu) return -1;
  if (bits == 8 && bf16) hipLaunchKernelGGL((aw_step_kernel<true, true>), dim3(grid), dim3(256), 0, stream, *a);
  else if (bits == 8) hipLaunchKernelGGL((aw_step_kernel<true, false>), dim3(grid), dim3(256), 0, stream, *a);
  else if (bf16) hipLaunchKernelGGL((aw_step_kernel<false, true>), dim3(grid), dim3(256), 0, stream, *a);
  else hipLaunchKernelGGL((aw_step_kernel<false, false>), dim3(grid), dim3(256), 0, stream, *a);
  return (int)hipGetLastError();
}

// grid: workgroups, one partial sum each
int rx_norm_part(const NormArgs* a, int grid, hipStream_t stream) {
  if (a->n <= 0 || a->n > kNormMax || grid <= 0) return -1;
  hipLaunchKernelGGL(norm_part_kernel, dim3((unsigned)grid), dim3(256), 0, stream, *a);
  return (int)hipGetLastError();
}

int rx_norm_scale(const ScaleArgs* a, int grid, hipStream_t stream) {
  if (a->t.n <= 0 || a->t.n > kNormMax || grid <= 0) return -1;
  hipLaunchKernelGGL(norm_scale_kernel, dim3((unsigned)grid), dim3(256), 0, stream, *a);
  return (int)hipGetLastError();
}

int rx_aw_decode(const uint8_t* m, const uint8_t* v, const uint8_t* sc, void* mo, void* vo, long long n, int bf16,
                 hipStream_t stream) {
  if (n <= 0) return 0;
  long long grid = (n + 1023) / 1024;
  grid = grid > 8192 ? 8192 : grid;
  if (bf16)
    hipLaunchKernelGGL((aw_decode_kernel<true>), dim3((unsigned)grid), dim3(256), 0, stream, m, v, sc, mo, vo, n);
  else
    hipLaunchKernelGGL((aw_decode_kernel<false>), dim3((unsigned)grid), dim3(256), 0, stream, m, v, sc, mo, vo, n);
  return (int)hipGetLastError();
}

}  // extern "C"
