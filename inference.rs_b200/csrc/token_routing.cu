// Tokens sorted by expert and back. A token has topk slots, each with the id of an expert; slots sorted by expert (those of one expert in
// their own order) are the rows that the experts' products run over.
//
//   position[slot] = row of the slot, -1 if its id is no expert's;   order[row] = slot;   rows of expert e: offsets[e] .. offsets[e + 1]
//   dispatch:  rows[position[t, j]] = x[t]                     its gradient:  dx[t] = sum_j drows[position[t, j]]
//   combine:   out[t] = sum_j weights[t, j] rows[position[t, j]]
//   gradients: drows[position[t, j]] = weights[t, j] dout[t],  dweights[t, j] = sum_i dout[t, i] rows[position[t, j], i]
//
// Everything is gathered or scattered by one owner of each output, in slot order and 32-bit sums: no atomics, the same bits every time.
#include "int8.cuh"

namespace b200q {

constexpr int RT_THREADS = 512;

// One CTA per expert, and one more for the slots of none. Each CTA counts by itself how many slots belong to experts before its own
// (its first row) and ranks its own slots, reading all ids twice: a few hundred KB out of L2 at most, where counting once and ranking
// afterwards would take two launches or CTAs that wait for one another.
template <typename Id>
__global__ void __launch_bounds__(RT_THREADS) route_sort_kernel(const Id* __restrict__ ids, int slots, int experts, int* __restrict__ order,
                                                               int* __restrict__ offsets, int* __restrict__ position) {
    __shared__ int before[RT_THREADS / 32 + 1], lower[RT_THREADS / 32];
    grid_launch_dependents();
    const int e = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int WARPS = RT_THREADS / 32;
    // a warp ranks a contiguous piece of the slots, 32 at a time
    const int piece = ((slots + WARPS - 1) / WARPS + 31) & ~31;
    const int from = min(warp * piece, slots), to = min(from + piece, slots);
    const auto expert_of = [&](int i) {
        const long long id = i < to ? (long long)ids[i] : -1;
        return id >= 0 && id < experts ? (int)id : experts;  // `experts`: of none
    };
    int mine = 0, less = 0;
    for (int i = from; i < to; i += 32) {
        const int id = expert_of(i + lane);
        mine += __popc(__ballot_sync(0xffffffffu, i + lane < to && id == e));
        less += __popc(__ballot_sync(0xffffffffu, i + lane < to && id < e));
    }
    if (lane == 0) {
        before[warp + 1] = mine;
        lower[warp] = less;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int sum = 0;
        for (int w = 0; w < WARPS; ++w) sum += lower[w];
        before[0] = sum;
        offsets[e] = sum;  // of e = experts: how many rows there are
        for (int w = 0; w < WARPS; ++w) before[w + 1] += before[w];
    }
    __syncthreads();
    int row = before[warp];
    for (int i = from; i < to; i += 32) {
        const bool is = i + lane < to && expert_of(i + lane) == e;
        const unsigned vote = __ballot_sync(0xffffffffu, is);
        if (is) {
            const int r = row + __popc(vote & ((1u << lane) - 1));
            position[i + lane] = e < experts ? r : -1;
            order[r] = e < experts ? i + lane : -1;
        }
        row += __popc(vote);
    }
}

cudaError_t route_sort(const void* ids, bool wide, int slots, int experts, int* order, int* offsets, int* position, cudaStream_t s) {
    const dim3 grid((unsigned)experts + 1, 1, 1);
    if (wide) return launch_kernel(route_sort_kernel<long long>, grid, RT_THREADS, 0, s, false, static_cast<const long long*>(ids), slots, experts, order, offsets, position);
    return launch_kernel(route_sort_kernel<int>, grid, RT_THREADS, 0, s, false, static_cast<const int*>(ids), slots, experts, order, offsets, position);
}

// V neighbouring values of a row, V = 1 or 16 bytes' worth of the narrowest type involved
template <typename T, int V> struct Values {
    float v[V];
    __device__ void load(const T* p) {
        if constexpr (V == 1) {
            v[0] = to_float<T>(*p);
        } else {
            alignas(16) T raw[V];
#pragma unroll
            for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) reinterpret_cast<uint4*>(raw)[i] = *(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = to_float<T>(raw[i]);
        }
    }
    __device__ void store(T* p) const {
        if constexpr (V == 1) {
            *p = from_float<T>(v[0]);
        } else {
            alignas(16) T raw[V];
#pragma unroll
            for (int i = 0; i < V; ++i) raw[i] = from_float<T>(v[i]);
#pragma unroll
            for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(raw)[i];
        }
    }
};
static bool rows_wide(const void* p, long long ld, int elem) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (elem == ELEM_F32 ? 4 : 2) % 16 == 0;
}

// A CTA per token reads it once and writes its rows; rows behind the last are zeroed by the CTA that they would have belonged to had no
// slot been left out.
template <typename U>
__global__ void __launch_bounds__(256) route_dispatch_kernel(const U* __restrict__ x, long long ldx, const int* __restrict__ position,
                                                             const int* __restrict__ valid, U* __restrict__ rows, int topk, int h) {
    const int t = blockIdx.x;
    const U* src = x + (long long)t * ldx;
    const int nvalid = min(*valid, (int)gridDim.x * topk);
    U zero{};
    for (int c = threadIdx.x; c < h; c += 256) {
        const U v = src[c];
        for (int j = 0; j < topk; ++j) {
            const long long r = (long long)t * topk + j;
            const int p = position[r];
            if (p >= 0 && p < nvalid) rows[(long long)p * h + c] = v;
            if (r >= nvalid) rows[r * h + c] = zero;
        }
    }
}

cudaError_t route_dispatch(int elem, const void* x, long long ldx, const int* position, const int* valid, void* rows, int tokens, int topk, int h,
                           cudaStream_t s) {
    const int es = elem == ELEM_F32 ? 4 : 2;
    const dim3 grid((unsigned)tokens, 1, 1);
    if (rows_wide(x, ldx, elem) && rows_wide(rows, h, elem))
        return launch_kernel(route_dispatch_kernel<uint4>, grid, 256, 0, s, false, static_cast<const uint4*>(x), ldx * es / 16, position, valid, static_cast<uint4*>(rows), topk, h * es / 16);
    if (es == 4) return launch_kernel(route_dispatch_kernel<uint32_t>, grid, 256, 0, s, false, static_cast<const uint32_t*>(x), ldx, position, valid, static_cast<uint32_t*>(rows), topk, h);
    return launch_kernel(route_dispatch_kernel<uint16_t>, grid, 256, 0, s, false, static_cast<const uint16_t*>(x), ldx, position, valid, static_cast<uint16_t*>(rows), topk, h);
}

// out[t] = sum_j weights[t, j] rows[position[t, j]]; weights null: 1.
template <typename In, typename Out, int V>
__global__ void __launch_bounds__(256) route_combine_kernel(const In* rows, long long ldr, const int* position, const float* weights, Out* out, int topk,
                                                            int h) {
    grid_dependency_wait();
    grid_launch_dependents();
    const long long t = blockIdx.x;
    for (int c = V * threadIdx.x; c < h; c += V * 256) {
        Values<Out, V> sum;
#pragma unroll
        for (int i = 0; i < V; ++i) sum.v[i] = 0.0f;
        for (int j = 0; j < topk; ++j) {
            const int p = position[t * topk + j];
            if (p < 0 || p >= (int)gridDim.x * topk) continue;
            const float w = weights != nullptr ? weights[t * topk + j] : 1.0f;
            Values<In, V> r;
            r.load(rows + p * ldr + c);
#pragma unroll
            for (int i = 0; i < V; ++i) sum.v[i] = fmaf(w, r.v[i], sum.v[i]);
        }
        sum.store(out + t * h + c);
    }
}

template <typename In, typename Out>
static cudaError_t combine_t(bool wide, const void* rows, long long ldr, const int* position, const float* weights, void* out, int tokens, int topk,
                             int h, cudaStream_t s, bool dependent) {
    const dim3 grid((unsigned)tokens, 1, 1);
    if (wide) return launch_kernel(route_combine_kernel<In, Out, 8>, grid, 256, 0, s, dependent, static_cast<const In*>(rows), ldr, position, weights, static_cast<Out*>(out), topk, h);
    return launch_kernel(route_combine_kernel<In, Out, 1>, grid, 256, 0, s, dependent, static_cast<const In*>(rows), ldr, position, weights, static_cast<Out*>(out), topk, h);
}
cudaError_t route_combine(int elem_in, int elem_out, const void* rows, long long ldr, const int* position, const float* weights, void* out,
                          int tokens, int topk, int h, cudaStream_t s, bool dependent) {
    const bool wide = h % 8 == 0 && rows_wide(rows, ldr, elem_in) && rows_wide(out, h, elem_out);
    if (elem_in == ELEM_F32) {
        if (elem_out == ELEM_F32) return combine_t<float, float>(wide, rows, ldr, position, weights, out, tokens, topk, h, s, dependent);
        if (elem_out == ELEM_F16) return combine_t<float, __half>(wide, rows, ldr, position, weights, out, tokens, topk, h, s, dependent);
        return combine_t<float, __nv_bfloat16>(wide, rows, ldr, position, weights, out, tokens, topk, h, s, dependent);
    }
    if (elem_in == ELEM_F16) {
        if (elem_out == ELEM_F32) return combine_t<__half, float>(wide, rows, ldr, position, weights, out, tokens, topk, h, s, dependent);
        if (elem_out == ELEM_F16) return combine_t<__half, __half>(wide, rows, ldr, position, weights, out, tokens, topk, h, s, dependent);
        return combine_t<__half, __nv_bfloat16>(wide, rows, ldr, position, weights, out, tokens, topk, h, s, dependent);
    }
    if (elem_out == ELEM_F32) return combine_t<__nv_bfloat16, float>(wide, rows, ldr, position, weights, out, tokens, topk, h, s, dependent);
    if (elem_out == ELEM_F16) return combine_t<__nv_bfloat16, __half>(wide, rows, ldr, position, weights, out, tokens, topk, h, s, dependent);
    return combine_t<__nv_bfloat16, __nv_bfloat16>(wide, rows, ldr, position, weights, out, tokens, topk, h, s, dependent);
}

// The gradients of combine, a CTA per token: its slots' rows of drows (each written by one CTA), and the products with the rows. Rows
// behind the last become zeros as in dispatch. Either output may be left out (null).
template <typename G, typename T, int V>
__global__ void __launch_bounds__(256) route_combine_grad_kernel(const G* __restrict__ grad_out, long long ldg, const T* __restrict__ rows, long long ldr,
                                                                 const int* __restrict__ position, const int* __restrict__ valid,
                                                                 const float* __restrict__ weights, T* __restrict__ grad_rows,
                                                                 float* __restrict__ grad_weights, int topk, int h) {
    __shared__ float part[8];
    const long long t = blockIdx.x;
    const int nvalid = min(*valid, (int)gridDim.x * topk), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int j = 0; j < topk; ++j) {
        const long long slot = t * topk + j;
        const int p = position[slot];
        float dot = 0.0f;
        if (p >= 0 && p < nvalid) {
            const float w = weights[slot];
            for (int c = V * threadIdx.x; c < h; c += V * 256) {
                Values<G, V> g;
                g.load(grad_out + t * ldg + c);
                if (grad_weights != nullptr) {
                    Values<T, V> r;
                    r.load(rows + p * ldr + c);
#pragma unroll
                    for (int i = 0; i < V; ++i) dot = fmaf(g.v[i], r.v[i], dot);
                }
                if (grad_rows != nullptr) {
                    Values<T, V> d;
#pragma unroll
                    for (int i = 0; i < V; ++i) d.v[i] = w * g.v[i];
                    d.store(grad_rows + (long long)p * h + c);
                }
            }
        }
        if (grad_rows != nullptr && slot >= nvalid) {
            Values<T, V> zero;
#pragma unroll
            for (int i = 0; i < V; ++i) zero.v[i] = 0.0f;
            for (int c = V * threadIdx.x; c < h; c += V * 256) zero.store(grad_rows + slot * h + c);
        }
        if (grad_weights != nullptr) {
            dot = warp_sum(dot);
            if (lane == 0) part[warp] = dot;
            __syncthreads();
            if (threadIdx.x == 0) {
                float sum = 0.0f;
                for (int i = 0; i < 8; ++i) sum += part[i];
                grad_weights[slot] = sum;
            }
            __syncthreads();
        }
    }
}

template <typename G, typename T>
static cudaError_t combine_grad_t(bool wide, const void* grad_out, long long ldg, const void* rows, long long ldr, const int* position, const int* valid,
                                  const float* weights, void* grad_rows, float* grad_weights, int tokens, int topk, int h, cudaStream_t s) {
    const dim3 grid((unsigned)tokens, 1, 1);
    const G* g = static_cast<const G*>(grad_out);
    const T* r = static_cast<const T*>(rows);
    T* d = static_cast<T*>(grad_rows);
    if (wide) return launch_kernel(route_combine_grad_kernel<G, T, 8>, grid, 256, 0, s, false, g, ldg, r, ldr, position, valid, weights, d, grad_weights, topk, h);
    return launch_kernel(route_combine_grad_kernel<G, T, 1>, grid, 256, 0, s, false, g, ldg, r, ldr, position, valid, weights, d, grad_weights, topk, h);
}
cudaError_t route_combine_grad(int elem_grad, int elem, const void* grad_out, long long ldg, const void* rows, long long ldr, const int* position,
                               const int* valid, const float* weights, void* grad_rows, float* grad_weights, int tokens, int topk, int h,
                               cudaStream_t s) {
    const bool wide = h % 8 == 0 && rows_wide(grad_out, ldg, elem_grad) && (grad_weights == nullptr || rows_wide(rows, ldr, elem)) &&
                      (grad_rows == nullptr || rows_wide(grad_rows, h, elem));
#define B200Q_GRAD(G, T) return combine_grad_t<G, T>(wide, grad_out, ldg, rows, ldr, position, valid, weights, grad_rows, grad_weights, tokens, topk, h, s)
    if (elem_grad == ELEM_F32) {
        if (elem == ELEM_F32) B200Q_GRAD(float, float);
        if (elem == ELEM_F16) B200Q_GRAD(float, __half);
        B200Q_GRAD(float, __nv_bfloat16);
    }
    if (elem_grad == ELEM_F16) {
        if (elem == ELEM_F32) B200Q_GRAD(__half, float);
        if (elem == ELEM_F16) B200Q_GRAD(__half, __half);
        B200Q_GRAD(__half, __nv_bfloat16);
    }
    if (elem == ELEM_F32) B200Q_GRAD(__nv_bfloat16, float);
    if (elem == ELEM_F16) B200Q_GRAD(__nv_bfloat16, __half);
    B200Q_GRAD(__nv_bfloat16, __nv_bfloat16);
#undef B200Q_GRAD
}

}  // namespace b200q
