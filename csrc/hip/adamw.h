// Arguments of csrc/hip/adamw.hip's entry points (shared with their callers in csrc/torch).
#pragma once
#include <stdint.h>

// One number for a list of sizes: both sides of the C interface compare what they were built with.
template <class... N>
constexpr unsigned long long rx_layout(N... sizes) {
  unsigned long long h = 1469598103934665603ull;      // FNV-1a
  for (const unsigned long long v : {(unsigned long long)sizes...}) h = (h ^ v) * 1099511628211ull;
  return h;
}

enum {
  kAwMax = 64,         // tensors in one step launch (kernel arguments under 4 KiB)
  kAwPrepMax = 256,    // tensors in one preparation launch (one thread each)
  kNormMax = 256,      // tensors in one norm / scale launch (kernel arguments under 4 KiB)
  kAwBlock = 256,      // elements that share a scale: 4 per lane of one wave
  kAwChunk = 2048,     // elements of a step workgroup: 4 waves, 2 scale blocks in flight in each
  kNormChunk = 8192,   // elements that a norm workgroup has in flight
  kNormGrid = 1024,    // workgroups, and so partial sums, of a norm launch at most
  kNormBf16 = 0x8000   // in NormArgs::last: the tensor is bf16
};

struct AwHead {        // one per launch group of a step
  float gscale;        // what gradients are multiplied with (clip factor, -1 to maximize)
  int skip;            // 1: the norm is not finite, the step is left out
};

struct AwTensor {      // what one step has in common for a tensor
  float nlr_bc1;       // -lr / (1 - b1^t)
  float decay;         // 1 - lr wd
  float rs_bc2;        // 1 / sqrt(1 - b2^t)
  uint32_t key;        // of its dither in this step
};

struct AwPrep {
  int n, maximize, npart, first;     // first: index of this launch's first tensor in tensors[]
  double lr, wd, b1, b2, max_norm;   // max_norm < 0: no clipping
  const float* lr_dev;               // not null: the learning rate, on the device
  const double* part;                // npart partial sums of squared gradients
  AwHead* head;
  AwTensor* tensors;
  float* norm;                       // not null: where the norm goes
  uint32_t seed, pad_;
  float* step[kAwPrepMax];           // the tensors' step words
  int ordinal[kAwPrepMax];           // their places in the optimizer
};

struct AwStep {
  int n, pad_;
  float b1, omb1, b2, omb2, eps, pad2_;
  const AwHead* head;
  const AwTensor* tensors;           // of this launch's first tensor
  void* p[kAwMax];
  const void* g[kAwMax];
  void* m[kAwMax];
  void* v[kAwMax];
  uint8_t* sc[kAwMax];               // [blocks][2] scale bytes (8-bit moments)
  uint16_t* img[kAwMax];             // bf16 image of an fp32 p (null: none)
  long long len[kAwMax];
  unsigned start[kAwMax + 1];        // first chunk of each tensor
};

struct NormArgs {
  int n, pad0_;
  double* part;                      // one partial sum per workgroup
  unsigned chunks, pad_;
  const void* g[kNormMax];
  unsigned start[kNormMax + 1];      // first chunk of each tensor
  uint16_t last[kNormMax];           // elements of its last chunk, and kNormBf16
};

static_assert(kNormChunk < kNormBf16, "a chunk's elements and the type share 16 bits");

struct ScaleArgs {
  NormArgs t;                        // t.part: the partial sums to finish
  int npart, pad_;
  double max_norm;
  float* norm;
};

constexpr unsigned long long kAwLayout =
    rx_layout(sizeof(AwHead), sizeof(AwTensor), sizeof(AwPrep), sizeof(AwStep), sizeof(NormArgs), sizeof(ScaleArgs), kAwMax,
              kAwPrepMax, kNormMax, kAwBlock, kAwChunk, kNormChunk, kNormGrid, kNormBf16);

extern "C" {
unsigned long long rx_aw_layout();
int rx_aw_prep(const AwPrep* a, void* stream);
// stream_past: the step's working set is larger than the last-level cache
int rx_aw_step(const AwStep* a, int bits, int bf16, int stream_past, void* stream);
// grid: workgroups, one partial sum each; stream_past: all gradients together are larger than the last-level cache
int rx_norm_part(const NormArgs* a, int grid, int stream_past, void* stream);
int rx_norm_scale(const ScaleArgs* a, int grid, int stream_past, void* stream);
// stream_past: codes and values take much of the last-level cache
int rx_aw_decode(const uint8_t* m, const uint8_t* v, const uint8_t* sc, void* mo, void* vo, long long n, int bf16,
                 int stream_past, void* stream);
}
