// Arguments of csrc/hip/experts.hip's entry points (shared with their callers in csrc/torch).
#pragma once
#include "hip/adamw.h"   // rx_layout

enum {
  kMaxExperts = 1024,
  kRouteMaxK = 32,
  kPlanThreads = 1024
};

struct PlanArgs {
  const void* ids;            // [n] int32, or int64 when wide
  int wide, n, E, chunk, blocks, capacity, rows, pad_;
  const int* counts;          // [blocks][E] (not used with one block)
  int* position;              // [n]
  int* source;                // [rows]
  int* load;                  // [E]
  int* offsets;               // [E + 1]
};

struct RowArgs {
  long long T, rows, ldx;     // samples, expert rows, elements between samples' rows (x)
  int k, D, lg, stream;       // lg: log2 of the lanes that work on a sample; stream: rows go past the caches
  const int* position;        // [T][k]
  const int* source;          // [rows]
  const void* x;              // scatter: samples' rows in; gather: not used
  const float* w;             // [T][k] or null
  const void* h;              // scatter: expert rows to take products with, or null; gather: expert rows in
  void* out;                  // scatter: expert rows out; gather: samples' rows out
  float* dw;                  // scatter with h: [T][k]
};

constexpr unsigned long long kExpertLayout =
    rx_layout(sizeof(PlanArgs), sizeof(RowArgs), kMaxExperts, kRouteMaxK, kPlanThreads);

// dtype: 0 fp32, 1 bf16, 2 fp16
extern "C" {
unsigned long long rx_expert_layout();
// norm: [T][2] peak and 1 / sum, written when not null
int rx_route_fwd(const void* z, long long ldz, int dtype, long long T, int E, int k, int renorm, float* w, int* ids,
                 float* norm, void* stream);
// norm null: softmax over the chosen ones (z is not read)
int rx_route_bwd(const void* z, long long ldz, int dtype, const float* norm, const float* w, const int* ids,
                 const float* dw, long long T, int E, int k, void* dz, void* stream);
// counts: blocks * E ints of scratch (not used with one block)
int rx_expert_plan(const PlanArgs* a, int* counts, void* stream);
int rx_rows_scatter(const RowArgs* a, int dtype, void* stream);
int rx_rows_gather(const RowArgs* a, int dtype, void* stream);
}
