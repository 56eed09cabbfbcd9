// The MXFP4 layer for a few tokens (mxfp4_few.hip) and the scratch allocator it shares with the general form.
#pragma once
#include "mxfp4_core.h"

namespace fr {

constexpr int kFewTokens = 32;  // columns of the matrix instruction
constexpr int kFewPairs = 256;  // routed pairs kept in LDS

// Consecutive 256-byte aligned pieces of a workspace; with a null base only their total counts.
struct MxBump {
  unsigned char* base;
  int64_t at = 0;
  template <typename T>
  T* take(int64_t count) {
    T* p = reinterpret_cast<T*>(reinterpret_cast<uintptr_t>(base) + static_cast<uintptr_t>(at));
    at = round_up(at + count * static_cast<int64_t>(sizeof(T)), 256);
    return p;
  }
};

// silu(g) u by exponential and reciprocal of the hardware, a unit in the last place each: the IEEE quotient is ten instructions of the gate/up
// epilogue's twenty-five per value.
__device__ __forceinline__ float mx_silu_mul(float g, float u) { return g * __builtin_amdgcn_rcpf(1.f + __expf(-g)) * u; }

struct MxFewScratch {
  float *topk_w, *parts;
  int32_t* ids;
  int* arrived;
  unsigned char *xq, *act;
};
bool mx_few_fits(int64_t M, int64_t F, int E, int topk);
int64_t mx_few_workspace(void* ws, int64_t M, int64_t H, int64_t F, int E, int topk, MxFewScratch* s);
int mx_few_layer(const void* x, int dtype, const void* w1, const void* w2, const void* logits, int logits_dtype, int64_t M, int64_t H,
                 int64_t F, int E, int topk, int renorm, void* out, void* workspace, hipStream_t st);

// linear_mxfp4 for few rows: whether it takes them, its workspace, the product
bool mx_few_linear_fits(int64_t M, int64_t N);
int64_t mx_few_linear_workspace(int64_t M, int64_t K);
int mx_few_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* w, int64_t N, void* out, void* workspace,
                  hipStream_t st);

}  // namespace fr
