// Attention of a batch of positions over an encoder's states: what its kernel families share.
#pragma once
#include "common.cuh"
#include "tensor_types.cuh"

namespace nnvb {

// A call's sizes, strides (elements) and pointers, as the kernels take them.
struct AttnArgs {
    int64_t qs[3], ks[3], vs[3], os[3], dos[3];    // batch, token, head
    const void *q, *k, *v, *dout;
    const void* o;                 // forward: written; backward: the forward call's output
    void* lse;
    const int32_t* lengths;
    void *dq, *dk, *dv;
    void* delta;                   // workspace: [B, Hq, Lq] sum_d dout * out (and the log-sum-exp beside it on the tensor cores)
    double scale;
    int B, Lq, Lk, Hq, Hkv, D;
    int dtype;
    int longest_first;             // few rows: batch entries in the order of their lengths
};

// valid states of batch entry b
__device__ __forceinline__ int attn_len(const AttnArgs& a, int b) {
    if (!a.lengths) return a.Lk;
    const int n = a.lengths[b];
    return n < 0 ? 0 : (n < a.Lk ? n : a.Lk);
}

__device__ __forceinline__ float exp_acc(float x) { return exp2f(x); }     // callers scale by log2(e)
__device__ __forceinline__ double exp_acc(double x) { return exp2(x); }
__device__ __forceinline__ float log_acc(float x) { return logf(x); }
__device__ __forceinline__ double log_acc(double x) { return log(x); }

constexpr int V_CHUNK = 64;                        // fp16 backward: states whose largest norm is kept

constexpr double LOG2E = 1.4426950408889634074;

// any type, head size up to 256, any strides
int attn_forward_simt(cudaStream_t st, const AttnArgs& a);
int attn_backward_simt(cudaStream_t st, const AttnArgs& a);
// up to eight rows (16-bit types: sixteen) a state head: positions times query heads sharing it; head size up to 128, 16-byte aligned rows
bool attn_rows_takes(const AttnArgs& a);
int attn_forward_rows(cudaStream_t st, const AttnArgs& a);
// float and double, head size up to 128
int attn_forward_wide(cudaStream_t st, const AttnArgs& a);
int attn_backward_wide(cudaStream_t st, const AttnArgs& a);      // needs attn_delta's result
// 16-bit types on the tensor cores; head size a multiple of 8 up to 128, 16-byte aligned rows
bool attn_tc_takes_forward(const AttnArgs& a);
int attn_forward_tc(cudaStream_t st, const AttnArgs& a);
bool attn_tc_takes_backward(const AttnArgs& a);
int attn_backward_tc(cudaStream_t st, const AttnArgs& a);
int attn_delta(cudaStream_t st, const AttnArgs& a);

}  // namespace nnvb
