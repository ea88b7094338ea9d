// Int8 rows with a scale each (weights: per output channel, activations: per token), their products, and the routing of tokens to
// experts: what the files of these operators share.
#pragma once
#include "common.cuh"
#include "runtime.h"

namespace b200q {

int set_error(int code, const char* msg);

// Sums of K products of at most 128 * 127 stay inside 32 bits up to here.
constexpr int INT8_MAX_K = 131072;
constexpr int INT8_MAX_EXPERTS = 1024;

// Activation of a gated product, act(gate) * up, by the ids of the reference's host side
// (crates/inference-quant/kernels/cuda/glu_activation.cuh:4-10); -1: the product is not gated.
enum Int8Act : int { INT8_ACT_NONE = -1, INT8_ACT_SILU = 0, INT8_ACT_GELU = 1, INT8_ACT_RELU = 2, INT8_ACT_GELU_ERF = 3, INT8_ACT_SIGMOID = 4 };
__device__ __forceinline__ float int8_activate(float x, int act) {
    switch (act) {
        case INT8_ACT_GELU: return 0.5f * x * (1.0f + tanhf(0.7978845608f * (x + 0.044715f * (x * x * x))));
        case INT8_ACT_RELU: return x > 0.0f ? x : (x <= 0.0f ? 0.0f : x);  // a NaN stays one
        case INT8_ACT_GELU_ERF: return 0.5f * x * (1.0f + erff(x * 0.70710678118654752440f));
        case INT8_ACT_SIGMOID: return 1.0f / (1.0f + expf(-x));
        default: return x / (1.0f + expf(-x));
    }
}

// A product of int8 rows: y[r][i] = (sum_k xq[r][k] wq[e][i][k]) * xs[r] * ws[e][i], where e is the expert whose rows [offsets[e],
// offsets[e + 1]) hold r (one matrix, all rows: offsets null). Gated: the matrix holds, of every 16 rows, 8 of gate and then 8 of up,
// and y has one column for a pair of them.
struct Int8Product {
    const int8_t* xq;  // [rows][ldx]
    const float* xs;
    const int8_t* wq;  // [experts * n][ldw]
    const float* ws;
    void* y;           // [rows][ldy]
    const int* offsets;
    int rows, n, k, ldx, ldw, experts, act;
    int n_out;         // columns of y: n, or, gated, the pairs that are real
    long long ldy;
    unsigned int* status;
};

template <typename Kern, typename... Args>
static cudaError_t launch_kernel(Kern kernel, dim3 grid, unsigned block, size_t smem, cudaStream_t s, bool dependent, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// int8_quantize.cu
cudaError_t int8_quantize_rows(int elem, const void* x, long long ldx, int8_t* q, long long ldq, float* scales, long long rows, int k,
                               const int* position, int topk, const int* row_limit, cudaStream_t s, bool dependent);
cudaError_t int8_dequantize_rows(int elem, const int8_t* q, long long ldq, const float* scales, void* out, long long rows, int k, cudaStream_t s);
// int8_rows.cu
cudaError_t int8_product_rows(int elem, const Int8Product& p, cudaStream_t s, bool dependent);
// int8_pair.cu
bool int8_pair_pays(const Int8Product& p);
int int8_product_pair(int elem, const Int8Product& p, cudaStream_t s, bool dependent);
// token_routing.cu
cudaError_t route_sort(const void* ids, bool wide, int slots, int experts, int* order, int* offsets, int* position, cudaStream_t s);
cudaError_t route_dispatch(int elem, const void* x, long long ldx, const int* position, const int* valid, void* rows, int tokens, int topk, int h,
                           cudaStream_t s);
cudaError_t route_combine(int elem_in, int elem_out, const void* rows, long long ldr, const int* position, const float* weights, void* out,
                          int tokens, int topk, int h, cudaStream_t s, bool dependent);
cudaError_t route_combine_grad(int elem_grad, int elem, const void* grad_out, long long ldg, const void* rows, long long ldr, const int* position,
                               const int* valid, const float* weights, void* grad_rows, float* grad_weights, int tokens, int topk, int h,
                               cudaStream_t s);

}  // namespace b200q
