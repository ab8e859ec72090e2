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
#include "adamw.h"
#include "rx_common.h"

namespace {

constexpr int kBlk = kAwBlock;

// dither: 2^32 / golden ratio and the fractional bits of sqrt(2), sqrt(3) as odd multipliers
constexpr uint32_t kPhi = 0x9E3779B1u, kSq2 = 0x6A09E667u, kSq3 = 0xBB67AE85u;

__device__ __forceinline__ uint32_t aw_mix(uint32_t x) {
  x = (x ^ (x >> 16)) * kSq2;
  x = (x ^ (x >> 15)) * kSq3;
  return x ^ (x >> 16);
}

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

// biased scale exponent of a block from the largest magnitude's bits without a sign (NaN and infinity: 255 or more)
__device__ __forceinline__ int aw_scale(uint32_t top) { return (int)((top + 0xFFFFFu) >> 23); }
__device__ __forceinline__ int aw_exp(int s) { return (s > 0 ? s : 1) - 127; }

// code <-> value: a value scaled so that the code's smallest normal lands on fp32's is a code in bits 20 on
constexpr int kMShift = 112, kVShift = 96;   // 126 - 14, 126 - 30
template <int Q>
__device__ __forceinline__ float aw_dec_m(uint32_t codes, int e) {   // byte Q: its sign goes to bit 31, the rest to 26..20
  const int c = (int)(codes << (24 - 8 * Q)) >> 24;
  return ldexpf(__uint_as_float((uint32_t)(c << 20) & 0x87F00000u), e + kMShift);
}
template <int Q>
__device__ __forceinline__ float aw_dec_v(uint32_t codes, int e) {
  return ldexpf(__uint_as_float(((codes >> (8 * Q)) & 0xFFu) << 20), e + kVShift);
}
// the code in the top byte
__device__ __forceinline__ uint32_t aw_enc_m(float m, int e, uint32_t rnd16) {
  const uint32_t a = __float_as_uint(ldexpf(fabsf(m), -e - kMShift)) + (rnd16 << 4) + 8u;
  return ((a << 4) & 0x7FFFFFFFu) | (__float_as_uint(m) & 0x80000000u);
}
__device__ __forceinline__ uint32_t aw_enc_v(float v, int e, uint32_t rnd16) {
  const uint32_t a = __float_as_uint(ldexpf(v, -e - kVShift)) + (rnd16 << 4) + 8u;
  return (v != 0.f ? max(a, 0x100000u) : a) << 4;      // what is not zero stays so: it is divided by
}
// the top bytes of four words
__device__ __forceinline__ uint32_t aw_pack(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0C0C0703u), hi = __builtin_amdgcn_perm(d, c, 0x07030C0Cu);
  return lo | hi;
}

// the upper half of x's bits plus the dither; two of them packed
__device__ __forceinline__ uint32_t aw_dither_bf16x2(float x, float y, uint32_t rx, uint32_t ry) {
  // (a NaN is made the plain one: its low bits plus the dither could carry into the sign)
  const uint32_t a = (x != x ? 0x7FC00000u : __float_as_uint(x)) + rx, b = (y != y ? 0x7FC00000u : __float_as_uint(y)) + ry;
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// Loads and stores of 4 consecutive elements from any address of the type's; n: how many there are (<= 4). Parameters and
// gradients may be slices of a larger buffer: gfx950 takes vectors at any element. NT: streamed past the caches. A step
// that touches more than the 256 MB of the last-level cache gains by that (24 M fp32 with 32-bit moments, 384 MB:
// 128 -> 112 us; 48 M with 8 bits: 148 -> 133), one that fits loses (16 M, 256 MB: 68 -> 76), so the host goes by the bytes.
typedef f32x4 __attribute__((aligned(4))) f32x4_u;
typedef rx_u32x2 __attribute__((aligned(2))) u32x2_u;
typedef u32x4 __attribute__((aligned(2))) u32x4_u;

template <bool NT, class T>
__device__ __forceinline__ T aw_get(const T* s) {
  if constexpr (NT) return __builtin_nontemporal_load(s);
  return *s;
}
template <bool NT, class T>
__device__ __forceinline__ void aw_put(T* s, T v) {
  if constexpr (NT) __builtin_nontemporal_store(v, s);
  else *s = v;
}

template <bool BF16, bool NT = false>
__device__ __forceinline__ f32x4 aw_load4(const void* base, long long i, int n) {
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if constexpr (BF16) {
    const u16* s = (const u16*)base + i;
    if (n == 4) {
      const rx_u32x2 w = aw_get<NT>((const u32x2_u*)s);
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
    if (n == 4) {
      r = aw_get<NT>((const f32x4_u*)s);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < n) r[k] = s[k];
    }
  }
  return r;
}

template <bool NT = false>
__device__ __forceinline__ void aw_store4(float* s, const f32x4& r, int n) {
  if (n == 4) {
    aw_put<NT>((f32x4_u*)s, (f32x4_u)r);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) s[k] = r[k];
  }
}
template <bool NT = false>
__device__ __forceinline__ void aw_store4h(u16* s, uint32_t lo, uint32_t hi, int n) {
  if (n == 4) {
    aw_put<NT>((u32x2_u*)s, (u32x2_u){lo, hi});
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) s[k] = (u16)((k < 2 ? lo : hi) >> (16 * (k & 1)));
  }
}
template <bool NT = false>
__device__ __forceinline__ uint32_t aw_load4c(const uint8_t* s, int n) {
  if (n == 4) return aw_get<NT>((const uint32_t*)s);
  uint32_t r = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < n) r |= (uint32_t)s[k] << (8 * k);
  return r;
}
template <bool NT = false>
__device__ __forceinline__ void aw_store4c(uint8_t* s, uint32_t c, int n) {
  if (n == 4) {
    aw_put<NT>((uint32_t*)s, c);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) s[k] = (uint8_t)(c >> (8 * k));
  }
}

__device__ __forceinline__ void aw_decode4(uint32_t mc, uint32_t vc, int sm, int sv, f32x4& m, f32x4& v) {
  const int em = aw_exp(sm), ev = aw_exp(sv);
  m[0] = aw_dec_m<0>(mc, em);
  m[1] = aw_dec_m<1>(mc, em);
  m[2] = aw_dec_m<2>(mc, em);
  m[3] = aw_dec_m<3>(mc, em);
  v[0] = aw_dec_v<0>(vc, ev);
  v[1] = aw_dec_v<1>(vc, ev);
  v[2] = aw_dec_v<2>(vc, ev);
  v[3] = aw_dec_v<3>(vc, ev);
}

constexpr int kStepUnroll = kAwChunk / (4 * kBlk);    // scale blocks of a wave that are in flight together

struct AwPlace {       // where a launch's workgroup works (wave-uniform)
  void* p;
  const void* g;
  void *m, *v;
  uint8_t* sc;
  u16* img;
  long long n;
};

// One lane's share of a scale block: 4 elements. FULL: the block lies inside the tensor, so loads and stores are
// whole and no lane branches; otherwise element by element under the tensor's end.
template <bool BITS8, bool BF16, bool NT, bool FULL>
struct AwLane {
  f32x4 p, g, m, v;
  uint32_t mc, vc;
  int sm, sv;

  __device__ __forceinline__ void load(const AwPlace& a, long long blk, long long i, int left) {
    p = aw_load4<BF16, NT>(a.p, i, left);
    g = aw_load4<BF16, NT>(a.g, i, left);
    if constexpr (BITS8) {
      const u16 s = *(const u16*)(a.sc + blk * 2);
      sm = s & 0xFF;
      sv = s >> 8;
      mc = aw_load4c<NT>((const uint8_t*)a.m + i, left);
      vc = aw_load4c<NT>((const uint8_t*)a.v + i, left);
    } else {
      m = aw_load4<false, NT>(a.m, i, left);
      v = aw_load4<false, NT>(a.v, i, left);
    }
  }

  __device__ __forceinline__ void step(const AwStep& c, const AwTensor& k, float gscale, const AwPlace& a, long long blk,
                                       long long i, int left, int lane) {
    float b1 = c.b1, b2 = c.b2;
    if constexpr (BITS8) {
      aw_decode4(mc, vc, sm, sv, m, v);
      // a block that was not finite: what remains of its moments is NaN
      b1 = sm == 255 ? __uint_as_float(0x7FC00000u) : b1;
      b2 = sv == 255 ? __uint_as_float(0x7FC00000u) : b2;
    }
    uint32_t h[4];
    uint32_t mtop = 0, vtop = 0;
    uint32_t x = 0;
    if constexpr (BITS8 || BF16) x = (uint32_t)i * kPhi + (uint32_t)((unsigned long long)i >> 32) * kSq2 + k.key;
    float root[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      {
#pragma clang fp contract(off)
        const float gq = g[q] * gscale;
        m[q] = b1 * m[q] + c.omb1 * gq;
        v[q] = b2 * v[q] + c.omb2 * (gq * gq);
      }
      root[q] = __builtin_amdgcn_sqrtf(v[q]);
    }
    // The instruction takes subnormals, whose roots are under 2^-63, for 0: nothing in a denominator with eps of 2^38 times
    // that (under half a step of it), an infinite update with eps = 0. (One branch for the launch's eps: 48 M bf16 with 8 bits
    // 101 -> 102 us; scaling every root 108, a second kernel path for such an eps 104.)
    if (__builtin_expect(c.eps < k.rs_bc2 * 0x1p-38f, 0)) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (v[q] < 0x1p-126f) root[q] = ldexpf(__builtin_amdgcn_sqrtf(ldexpf(v[q], 32)), -16);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // square root and quotient to 1 ulp each: the update is about 1e-3 of p
      const float den = fmaf(root[q], k.rs_bc2, c.eps);
      p[q] = fmaf(k.nlr_bc1, m[q] * __builtin_amdgcn_rcpf(den), p[q] * k.decay);
      if (FULL || q < left) {
        mtop = max(mtop, __float_as_uint(m[q]) & 0x7FFFFFFFu);
        vtop = max(vtop, __float_as_uint(v[q]));       // (a NaN's sign: the largest of all)
      }
      // (a lane's 4 indexes do not cross 2^32)
      if constexpr (BITS8 || BF16) h[q] = aw_mix(x + q * kPhi);
    }
    if constexpr (BITS8) {
      const int sm1 = aw_scale(aw_wavemax(mtop)), sv1 = aw_scale(aw_wavemax(vtop) & 0x7FFFFFFFu);
      const int em = aw_exp(sm1), ev = aw_exp(sv1);
      uint32_t me[4], ve[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        me[q] = aw_enc_m(m[q], em, h[q] & 0xFFFFu);
        ve[q] = aw_enc_v(v[q], ev, h[q] >> 16);
      }
      const uint32_t m1 = sm1 >= 255 ? 0u : aw_pack(me[0], me[1], me[2], me[3]);
      const uint32_t v1 = sv1 >= 255 ? 0u : aw_pack(ve[0], ve[1], ve[2], ve[3]);
      aw_store4c<NT>((uint8_t*)a.m + i, m1, left);
      aw_store4c<NT>((uint8_t*)a.v + i, v1, left);
      if (lane == 0) *(u16*)(a.sc + blk * 2) = (u16)(min(sm1, 255) | min(sv1, 255) << 8);
    } else {
      aw_store4<NT>((float*)a.m + i, m, left);
      aw_store4<NT>((float*)a.v + i, v, left);
    }
    if constexpr (BF16) {
      // no master copy: rounded with the dither, so that updates under half a step of p are not lost
      const uint32_t lo = aw_dither_bf16x2(p[0], p[1], (h[0] * kSq2) >> 16, (h[1] * kSq2) >> 16);
      const uint32_t hi = aw_dither_bf16x2(p[2], p[3], (h[2] * kSq2) >> 16, (h[3] * kSq2) >> 16);
      aw_store4h<NT>((u16*)a.p + i, lo, hi, left);
    } else {
      aw_store4<NT>((float*)a.p + i, p, left);
      if (a.img != nullptr) {
        aw_store4h(a.img + i, rx_f2bf2(p[0], p[1]), rx_f2bf2(p[2], p[3]), left);
      }
    }
  }
};

// Bound by memory: 16 bytes an element with 8-bit moments and fp32 parameters, 10 with bf16 ones, 28 and 22 with 32-bit
// moments; one pass, a workgroup per 2048 elements of one tensor (found by bisection over at most 64 starts). A scale block
// is one wave's 4 elements a lane, so its two maxima are six lane exchanges in registers; two blocks per wave are loaded
// before the first is worked on (bf16: 104 -> 99 us for 48 M; four give nothing more). Coding, dither and update are about 65
// issue slots an element, of the 76 that bf16 leaves per element at 5 TB/s: they had to come down from 90 (bytes packed
// by v_perm, m's code decoded by one sign-extending shift, square root and reciprocal to 1 ulp). 35.4 M fp32 in 17 tensors:
// 92 us with 8 bits (6.1 TB/s), 161 us with 32 (6.1); bf16: 16.8 M in 64 tensors with 8 bits 36 us (4.6), 50.3 M in 3 with 32
// bits 178 us (6.2).
template <bool BITS8, bool BF16, bool NT>
__global__ __launch_bounds__(256) void aw_step_kernel(AwStep c) {
  const AwHead head = *c.head;
  if (head.skip) return;
  const int t = aw_find(c, c.n, blockIdx.x);
  const AwTensor k = c.tensors[t];
  const AwPlace a = {c.p[t], c.g[t], c.m[t], c.v[t], BITS8 ? c.sc[t] : nullptr, BF16 ? nullptr : c.img[t], c.len[t]};
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long blk = ((long long)(blockIdx.x - c.start[t]) * 4 + wave) * kStepUnroll;
  if ((blk + kStepUnroll) * kBlk <= a.n) {
    AwLane<BITS8, BF16, NT, true> w[kStepUnroll];
#pragma unroll
    for (int u = 0; u < kStepUnroll; ++u) w[u].load(a, blk + u, (blk + u) * kBlk + lane * 4, 4);
#pragma unroll
    for (int u = 0; u < kStepUnroll; ++u) w[u].step(c, k, head.gscale, a, blk + u, (blk + u) * kBlk + lane * 4, 4, lane);
    return;
  }
  for (long long b = blk; b < blk + kStepUnroll && b * kBlk < a.n; ++b) {
    const long long i = b * kBlk + lane * 4;
    const int left = a.n - i >= 4 ? 4 : a.n - i > 0 ? (int)(a.n - i) : 0;
    AwLane<BITS8, BF16, NT, false> w;
    w.load(a, b, i, left);
    w.step(c, k, head.gscale, a, b, i, left, lane);
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

// (a launch gives up to 1024 partial sums: 4 loads a thread, in flight together)
__device__ __forceinline__ double aw_partsum(const double* part, int npart, double* lds) {
  double s = 0.0;
  for (int i0 = 0; i0 < npart; i0 += kNormGrid) {
    double v[kNormGrid / 256];
#pragma unroll
    for (int u = 0; u < kNormGrid / 256; ++u) {
      const int i = i0 + u * 256 + (int)threadIdx.x;
      v[u] = i < npart ? part[i] : 0.0;
    }
#pragma unroll
    for (int u = 0; u < kNormGrid / 256; ++u) s += v[u];
  }
  return aw_blocksum(s, lds);
}

// b^n by squaring: under 50 products, each to half an ulp of 64 bits
__device__ __forceinline__ double aw_pow(double b, uint32_t n) {
  double r = 1.0;
  for (; n != 0; n >>= 1) {
    if (n & 1) r *= b;
    b *= b;
  }
  return r;
}

// min(1, max / (norm + 1e-6)): the factor of torch.nn.utils.clip_grad_norm_
__device__ __forceinline__ float aw_clip(double norm, double max_norm) {
  const double c = max_norm / (norm + 1e-6);
  return (float)(c < 1.0 ? c : c >= 1.0 ? 1.0 : c);   // (a NaN stays one)
}

// One workgroup, a thread per tensor: latency only (3.0 us for 18 tensors, 4.4 for 192 and 1500 partial sums). It could be
// part of the step's workgroups but for the step words, which all of them would read while one counts them on.
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
  const uint32_t t = (uint32_t)step;
  const double lr = a.lr_dev != nullptr ? (double)*a.lr_dev : a.lr;
  AwTensor k;
  k.nlr_bc1 = (float)(-lr / (1.0 - aw_pow(a.b1, t)));
  k.decay = (float)(1.0 - lr * a.wd);
  k.rs_bc2 = (float)(1.0 / sqrt(1.0 - aw_pow(a.b2, t)));
  k.key = aw_mix(aw_mix(a.seed + (uint32_t)a.ordinal[i] * kPhi) + t);
  a.tensors[a.first + i] = k;
}

// Sums of squares in 64 bits: the norm then does not depend on the order of the sum in any of its 32 bits but by chance.
// Bound by memory (a conversion and a 64-bit multiply-add an element fit beside it): 8192 elements are loaded before the
// first is squared, 1024 workgroups give 16 waves a CU. 50 M fp32 in 36 us (5.6 TB/s; 4096 elements: 38, 512 workgroups: 52),
// bf16 in 20; 67 M fp32 in 256 tensors, streamed, 43 us, and 3.8 for a scaling that finds a factor of 1
// (with 128 tensors a launch: 55 in all).
// 4 x 4 (bf16: 2 x 8) elements of a lane, in flight together
template <bool BF16, bool FULL, bool NT>
__device__ __forceinline__ double aw_squares(const void* g, long long i, long long n) {
  double s = 0.0;
  if constexpr (BF16 && FULL) {
    u32x4 w[kNormChunk / 2048];
#pragma unroll
    for (int u = 0; u < kNormChunk / 2048; ++u) w[u] = aw_get<NT>((const u32x4_u*)((const u16*)g + i + u * 2048 + threadIdx.x * 8));
#pragma unroll
    for (int u = 0; u < kNormChunk / 2048; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float a = __uint_as_float(w[u][q] << 16), b = __uint_as_float(w[u][q] & 0xFFFF0000u);
        s = fma((double)a, (double)a, s);
        s = fma((double)b, (double)b, s);
      }
    return s;
  }
  f32x4 v[kNormChunk / 1024];
#pragma unroll
  for (int u = 0; u < kNormChunk / 1024; ++u) {
    const long long j = i + u * 1024 + threadIdx.x * 4;
    v[u] = aw_load4<BF16, NT>(g, j, FULL ? 4 : n - j >= 4 ? 4 : n - j > 0 ? (int)(n - j) : 0);
  }
#pragma unroll
  for (int u = 0; u < kNormChunk / 1024; ++u)
#pragma unroll
    for (int q = 0; q < 4; ++q) s = fma((double)v[u][q], (double)v[u][q], s);
  return s;
}

// elements of chunk c, which is one of tensor t's
__device__ __forceinline__ int norm_count(const NormArgs& a, int t, unsigned c) {
  return c + 1 < a.start[t + 1] ? (int)kNormChunk : (int)(a.last[t] & ~kNormBf16);
}

// a workgroup takes consecutive chunks, so that it looks for its tensor once and then walks on
template <bool NT>
__global__ __launch_bounds__(256) void norm_part_kernel(NormArgs a) {
  __shared__ double lds[4];
  double s = 0.0;
  const unsigned per = a.chunks / gridDim.x, more = a.chunks % gridDim.x, b = blockIdx.x;
  const unsigned first = b * per + min(b, more), last = first + per + (b < more ? 1u : 0u);
  int t = first < last ? aw_find(a, a.n, first) : 0;
  for (unsigned c = first; c < last; ++c) {
    while (c >= a.start[t + 1]) ++t;
    const void* g = a.g[t];
    const long long i = (long long)(c - a.start[t]) * kNormChunk, n = i + norm_count(a, t, c);
    const bool full = n == i + kNormChunk;
    if (a.last[t] & kNormBf16) s += full ? aw_squares<true, true, NT>(g, i, n) : aw_squares<true, false, NT>(g, i, n);
    else s += full ? aw_squares<false, true, NT>(g, i, n) : aw_squares<false, false, NT>(g, i, n);
  }
  s = aw_blocksum(s, lds);
  if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

template <bool BF16, bool FULL, bool NT>
__device__ __forceinline__ void aw_scale_chunk(void* g, long long i, long long n, float f) {
  constexpr int U = kNormChunk / 1024;
  f32x4 v[U];
  int left[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long j = i + u * 1024 + threadIdx.x * 4;
    left[u] = FULL ? 4 : n - j >= 4 ? 4 : n - j > 0 ? (int)(n - j) : 0;
    v[u] = aw_load4<BF16, NT>(g, j, left[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long j = i + u * 1024 + threadIdx.x * 4;
    v[u] *= f;
    if constexpr (BF16) aw_store4h<NT>((u16*)g + j, rx_f2bf2(v[u][0], v[u][1]), rx_f2bf2(v[u][2], v[u][3]), left[u]);
    else aw_store4<NT>((float*)g + j, v[u], left[u]);
  }
}

// 67 M in 64 tensors, norm and scaling: fp32 157 us streamed, 172 through the caches (three passes over 268 MB); bf16 86, 97.
// g *= min(1, max_norm / (norm + 1e-6)); every workgroup finishes the norm itself (a few KB out of L2), which saves a
// launch between the two passes; with a factor of 1 nothing is touched
template <bool NT>
__global__ __launch_bounds__(256) void norm_scale_kernel(ScaleArgs a) {
  __shared__ double lds[4];
  const double norm = sqrt(aw_partsum(a.t.part, a.npart, lds));
  const float f = aw_clip(norm, a.max_norm);
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.norm != nullptr) *a.norm = (float)norm;
  if (f == 1.f) return;
  const unsigned per = a.t.chunks / gridDim.x, more = a.t.chunks % gridDim.x, b = blockIdx.x;
  const unsigned first = b * per + min(b, more), last = first + per + (b < more ? 1u : 0u);
  int t = first < last ? aw_find(a.t, a.t.n, first) : 0;
  for (unsigned c = first; c < last; ++c) {
    while (c >= a.t.start[t + 1]) ++t;
    void* g = const_cast<void*>(a.t.g[t]);
    const long long i = (long long)(c - a.t.start[t]) * kNormChunk, n = i + norm_count(a.t, t, c);
    const bool full = n == i + kNormChunk;
    if (a.t.last[t] & kNormBf16) full ? aw_scale_chunk<true, true, NT>(g, i, n, f) : aw_scale_chunk<true, false, NT>(g, i, n, f);
    else full ? aw_scale_chunk<false, true, NT>(g, i, n, f) : aw_scale_chunk<false, false, NT>(g, i, n, f);
  }
}

// codes -> the values they stand for (at most 4 significant bits: exact in bf16 too); a wave takes whole scale blocks, four
// of them in flight. Bound by memory: 35.4 M to bf16 in 37 us (5.7 TB/s)
constexpr int kDecUnroll = 4;

template <bool BF16, bool NT>
__device__ __forceinline__ void aw_decode_store(uint32_t mc, uint32_t vc, uint32_t s, void* mo, void* vo, long long i,
                                                int left) {
  const int sm = s & 0xFF, sv = s >> 8;
  f32x4 m, v;
  aw_decode4(mc, vc, sm, sv, m, v);
  const float nan = __uint_as_float(0x7FC00000u);
  if (sm == 255) m = (f32x4){nan, nan, nan, nan};
  if (sv == 255) v = (f32x4){nan, nan, nan, nan};
  if constexpr (BF16) {
    aw_store4h<NT>((u16*)mo + i, rx_f2bf2(m[0], m[1]), rx_f2bf2(m[2], m[3]), left);
    aw_store4h<NT>((u16*)vo + i, rx_f2bf2(v[0], v[1]), rx_f2bf2(v[2], v[3]), left);
  } else {
    aw_store4<NT>((float*)mo + i, m, left);
    aw_store4<NT>((float*)vo + i, v, left);
  }
}

template <bool BF16, bool NT>
__global__ __launch_bounds__(256) void aw_decode_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ v,
                                                        const uint8_t* __restrict__ sc, void* __restrict__ mo,
                                                        void* __restrict__ vo, long long n) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long blk = ((long long)blockIdx.x * 4 + wave) * kDecUnroll;
  if ((blk + kDecUnroll) * kBlk <= n) {
    uint32_t mc[kDecUnroll], vc[kDecUnroll], s[kDecUnroll];
#pragma unroll
    for (int u = 0; u < kDecUnroll; ++u) {
      s[u] = *(const u16*)(sc + (blk + u) * 2);
      mc[u] = aw_get<NT>((const uint32_t*)(m + (blk + u) * kBlk + lane * 4));
      vc[u] = aw_get<NT>((const uint32_t*)(v + (blk + u) * kBlk + lane * 4));
    }
#pragma unroll
    for (int u = 0; u < kDecUnroll; ++u)
      aw_decode_store<BF16, NT>(mc[u], vc[u], s[u], mo, vo, (blk + u) * kBlk + lane * 4, 4);
    return;
  }
  for (long long b = blk; b < blk + kDecUnroll && b * kBlk < n; ++b) {
    const long long i = b * kBlk + lane * 4;
    const int left = n - i >= 4 ? 4 : n - i > 0 ? (int)(n - i) : 0;
    aw_decode_store<BF16, NT>(aw_load4c(m + i, left), aw_load4c(v + i, left), *(const u16*)(sc + b * 2), mo, vo, i, left);
  }
}

}  // namespace

extern "C" {

unsigned long long rx_aw_layout() { return kAwLayout; }

int rx_aw_prep(const AwPrep* a, void* on) {
  hipStream_t stream = static_cast<hipStream_t>(on);
  if (a->n < 0 || a->n > kAwPrepMax) return -1;
  hipLaunchKernelGGL(aw_prep_kernel, dim3(1), dim3(256), 0, stream, *a);
  return (int)hipGetLastError();
}

int rx_aw_step(const AwStep* a, int bits, int bf16, int stream_past, void* on) {
  hipStream_t stream = static_cast<hipStream_t>(on);
  if (a->n <= 0 || a->n > kAwMax || (bits != 8 && bits != 32)) return -1;
  const unsigned grid = a->start[a->n];
  if (grid == 0) return 0;
  if (grid > 0x7FFFFFFFu) return -1;
#define RX_AW(BITS8, BF16)                                                                                             \
  do {                                                                                                                 \
    if (stream_past) hipLaunchKernelGGL((aw_step_kernel<BITS8, BF16, true>), dim3(grid), dim3(256), 0, stream, *a);    \
    else hipLaunchKernelGGL((aw_step_kernel<BITS8, BF16, false>), dim3(grid), dim3(256), 0, stream, *a);               \
  } while (0)
  if (bits == 8 && bf16) RX_AW(true, true);
  else if (bits == 8) RX_AW(true, false);
  else if (bf16) RX_AW(false, true);
  else RX_AW(false, false);
#undef RX_AW
  return (int)hipGetLastError();
}

int rx_norm_part(const NormArgs* a, int grid, int stream_past, void* on) {
  hipStream_t stream = static_cast<hipStream_t>(on);
  if (a->n <= 0 || a->n > kNormMax || grid <= 0) return -1;
  if (stream_past) hipLaunchKernelGGL(norm_part_kernel<true>, dim3((unsigned)grid), dim3(256), 0, stream, *a);
  else hipLaunchKernelGGL(norm_part_kernel<false>, dim3((unsigned)grid), dim3(256), 0, stream, *a);
  return (int)hipGetLastError();
}

int rx_norm_scale(const ScaleArgs* a, int grid, int stream_past, void* on) {
  hipStream_t stream = static_cast<hipStream_t>(on);
  if (a->t.n <= 0 || a->t.n > kNormMax || grid <= 0) return -1;
  if (stream_past) hipLaunchKernelGGL(norm_scale_kernel<true>, dim3((unsigned)grid), dim3(256), 0, stream, *a);
  else hipLaunchKernelGGL(norm_scale_kernel<false>, dim3((unsigned)grid), dim3(256), 0, stream, *a);
  return (int)hipGetLastError();
}

int rx_aw_decode(const uint8_t* m, const uint8_t* v, const uint8_t* sc, void* mo, void* vo, long long n, int bf16,
                 int stream_past, void* on) {
  hipStream_t stream = static_cast<hipStream_t>(on);
  if (n <= 0) return 0;
  const long long grid = (n + 4 * kDecUnroll * kBlk - 1) / (4 * kDecUnroll * kBlk);
  if (grid > 0x7FFFFFFFll) return -1;
#define RX_DECODE(BF16, NT) \
  hipLaunchKernelGGL((aw_decode_kernel<BF16, NT>), dim3((unsigned)grid), dim3(256), 0, stream, m, v, sc, mo, vo, n)
  if (bf16 && stream_past) RX_DECODE(true, true);
  else if (bf16) RX_DECODE(true, false);
  else if (stream_past) RX_DECODE(false, true);
  else RX_DECODE(false, false);
#undef RX_DECODE
  return (int)hipGetLastError();
}

}  // extern "C"
