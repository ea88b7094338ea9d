// Int8 rows with a scale each (weights: per output channel, activations: per token), their products, and the routing of tokens to
// experts: what the files of these operators share.
#pragma once
#include "common.cuh"
#include "runtime.h"

namespace b200q {

int set_error(int code, const char* msg);

// Sums of K products of at most 128 * 128 stay inside 32 bits up to here.
constexpr int INT8_MAX_K = 131071;
constexpr int INT8_MAX_EXPERTS = 1024;

// Activation of a gated product, act(gate) * up, by the ids of the reference's host side
// (crates/inference-quant/kernels/cuda/glu_activation.cuh:4-10); -1: the product is not gated.
enum Int8Act : int { INT8_ACT_NONE = -1, INT8_ACT_SILU = 0, INT8_ACT_GELU = 1, INT8_ACT_RELU = 2, INT8_ACT_GELU_ERF = 3, INT8_ACT_SIGMOID = 4 };
// x / (1 + exp(-t)) without a branch, its error in proportion to its size everywhere: exp(-|t|) neither overflows nor cancels, and the
// reciprocal is one of 1 to 2. Two units of the last place for the exponential, one for the reciprocal, half of one for each other
// rounding (for t below -87, where the exponential is subnormal, 2^-148 |x|). The layer of 2048 tokens through 2 of 8 experts of 4096 x
// 14336 takes 620 us (708 at the power cap); 612 (700) with ex2.approx of -t log2(e) and rcp.approx of 1 + exp(-t), which are off by
// |t| 2^-24 below zero and give 0 from -87 on; 720 at the cap with a Newton step on the reciprocal.
__device__ __forceinline__ float times_sigmoid(float x, float t) {
    const float e = expf(-fabsf(t)), d = 1.0f + e;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return (t < 0.0f ? x * e : x) * r;
}
__device__ __forceinline__ float int8_activate(float x, int act) {
    switch (act) {
        case INT8_ACT_GELU: return times_sigmoid(x, 1.5957691216f * (x + 0.044715f * (x * x * x)));  // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u))
        case INT8_ACT_RELU: return x > 0.0f ? x : (x <= 0.0f ? 0.0f : x);  // a NaN stays one
        case INT8_ACT_GELU_ERF: return 0.5f * x * (1.0f + erff(x * 0.70710678118654752440f));
        case INT8_ACT_SIGMOID: return times_sigmoid(1.0f, x);
        default: return times_sigmoid(x, x);
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
    // offsets are older than the launch before this one, which lets this one begin only when it has waited for all before it: they are
    // read (out of L2) and the first weights asked for without a wait (experts' layer, 1 token through 2 of 8 experts of 4096 x 14336
    // 67.8 -> 66.2 us, 1024 through 8 of 128 of 2048 x 768 157.3 -> 152.0)
    bool offsets_known;
    const void* ids;  // the slots' expert ids, from which a CTA finds the offsets by itself, known as they are (null: it reads them)
    bool wide_ids;
};

__device__ __forceinline__ int expert_id(const void* ids, bool wide, int experts, int slot) {  // `experts`: of none
    const long long id = wide ? static_cast<const long long*>(ids)[slot] : static_cast<const int*>(ids)[slot];
    return id >= 0 && id < experts ? (int)id : experts;
}
// Where the experts' rows begin, from the slots' ids, by all threads of a CTA: off[0 .. experts] in shared memory. (Out of line: in line, its
// instructions cost the products that do not call it 0.6 us.)
static __device__ __noinline__ void expert_offsets(const void* ids, bool wide, int experts, int slots, int* off) {
    for (int e = threadIdx.x; e <= experts; e += blockDim.x) off[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < slots; i += blockDim.x) {
        const int e = expert_id(ids, wide, experts, i);
        if (e < experts) atomicAdd(&off[e], 1);  // (integers: any order)
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        int sum = 0;
        for (int e0 = 0; e0 <= experts; e0 += 32) {
            const int e = e0 + threadIdx.x, c = e < experts ? off[e] : 0;
            int upto = c;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const int v = __shfl_up_sync(0xffffffffu, upto, d);
                if ((int)threadIdx.x >= d) upto += v;
            }
            if (e <= experts) off[e] = sum + upto - c;
            sum += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    __syncthreads();
}

// Where a tile of a product lies: its weight tile, its expert, its tokens.
struct Int8Tile {
    int tn, e, row0, toks;
};
// The tiles of all experts as one list: of up to `bn` tokens of one expert each, the tokens of a weight tile one after the other.
inline constexpr size_t int8_list_bytes(int experts) { return experts > 1 ? 8 * (size_t)(experts + 1) + 128 : 0; }
struct Int8TileList {
    const int* start;    // shared memory: tiles before each expert's, experts + 1 of them (null: one matrix)
    const int* offsets;  // shared memory
    int experts, row0, rows, bn, tiles_n, ntiles, at;

    // by all threads of a CTA; `shared`: int8_list_bytes
    template <int THREADS> __device__ __forceinline__ void build(const Int8Product& p, int bn_, int tiles_n_, int* shared) {
        start = offsets = nullptr;
        experts = p.experts;
        row0 = 0;
        rows = p.rows;
        bn = bn_;
        tiles_n = tiles_n_;
        at = 0;
        if (p.offsets != nullptr && !p.offsets_known) grid_dependency_wait();  // where the experts' rows begin is the work of a launch before
        if (experts == 1) {
            if (p.offsets != nullptr) {
                row0 = min(max(__ldcg(p.offsets), 0), p.rows);
                rows = max(min(__ldcg(p.offsets + 1), p.rows) - row0, 0);
            }
            ntiles = (rows + bn - 1) / bn * tiles_n;
            return;
        }
        const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
        int *scan = shared, *off = shared + 32, *st = off + experts + 1;
        if (p.ids != nullptr) {
            expert_offsets(p.ids, p.wide_ids, experts, p.rows, off);
        } else {
            for (int i = tid; i <= experts; i += THREADS) off[i] = min(max(__ldcg(p.offsets + i), 0), p.rows);
            __syncthreads();
        }
        const int per = (experts + THREADS - 1) / THREADS, e0 = tid * per, e1 = min(e0 + per, experts);
        int sum = 0;
        for (int e = e0; e < e1; ++e) sum += (max(off[e + 1] - off[e], 0) + bn - 1) / bn * tiles_n;
        int upto = sum;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
        }
        if (lane == 31) scan[warp] = upto;
        __syncthreads();
        int before = upto - sum;
        for (int w = 0; w < warp; ++w) before += scan[w];
        for (int e = e0; e < e1; ++e) {
            st[e] = before;
            before += (max(off[e + 1] - off[e], 0) + bn - 1) / bn * tiles_n;
            if (e == experts - 1) st[experts] = before;
        }
        __syncthreads();
        start = st;
        offsets = off;
        ntiles = st[experts];
    }
    // by whole warps, with tiles that do not fall
    __device__ __forceinline__ Int8Tile find(int tile, int lane) {
        Int8Tile t;
        int first = row0, count = rows;
        t.e = 0;
        if (start != nullptr) {
            for (;; at += 32) {
                const int i = at + lane + 1;
                const unsigned above = __ballot_sync(0xffffffffu, i > experts || start[i] > tile);
                if (above != 0) {
                    t.e = at + __ffs(above) - 1;
                    break;
                }
            }
            tile -= start[t.e];
            first = offsets[t.e];
            count = offsets[t.e + 1] - first;
        }
        // an expert's tiles are of one height but for the last, where the instruction's steps of 32 tokens allow it; never above bn
        const int tiles_m = (count + bn - 1) / bn, height = bn % 32 == 0 ? min(bn, ((count + tiles_m - 1) / tiles_m + 31) & ~31) : bn;
        t.tn = tile / tiles_m;
        const int tm = tile - t.tn * tiles_m;
        t.row0 = first + tm * height;
        t.toks = min(height, count - tm * height);
        return t;
    }
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
bool int8_routes_quantizing(int tokens, int topk, int k);
cudaError_t int8_route_quantize(int elem, const void* x, long long ldx, int8_t* q, long long ldq, float* scales, int tokens, int k, const void* ids,
                                bool wide_ids, int topk, int experts, int* position, int* offsets, cudaStream_t s);
cudaError_t int8_dequantize_rows(int elem, const int8_t* q, long long ldq, const float* scales, void* out, long long rows, int k, cudaStream_t s);
// int8_rows.cu
bool int8_rows_pays(const Int8Product& p);
cudaError_t int8_product_rows(int elem, const Int8Product& p, cudaStream_t s, bool dependent);
// int8_pair.cu
bool int8_pair_ready();
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
