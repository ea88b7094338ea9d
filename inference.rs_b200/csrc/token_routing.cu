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

constexpr int RT_THREADS = 1024;
constexpr int RT_HELD = 8;      // ids that a lane reads at once
constexpr int RT_ROW_THREADS = 256;
constexpr int RT_ROW_CTAS = 8;  // CTAs of as many threads on an SM

// One CTA per expert, and one more for the slots of none. Each CTA counts by itself how many slots belong to experts before its own
// (its first row) and ranks its own slots, reading all ids twice: a few hundred KB out of L2 at most, where counting once and ranking
// afterwards would take two launches or CTAs that wait for one another. Up to 8192 slots a warp's ids stay in registers in between.
template <typename Id>
__global__ void __launch_bounds__(RT_THREADS) route_sort_kernel(const Id* __restrict__ ids, int slots, int experts, int* __restrict__ order,
                                                               int* __restrict__ offsets, int* __restrict__ position) {
    constexpr int WARPS = RT_THREADS / 32, CHUNK = 32 * RT_HELD;
    __shared__ int before[WARPS], lower[WARPS];
    grid_launch_dependents();
    const int e = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a warp ranks a contiguous piece of the slots
    const int piece = ((slots + WARPS - 1) / WARPS + CHUNK - 1) / CHUNK * CHUNK;
    const int from = (int)min((long long)warp * piece, (long long)slots), to = min(from + piece, slots);
    int held[RT_HELD];
    const auto read = [&](int i) {
        Id raw[RT_HELD];
#pragma unroll
        for (int j = 0; j < RT_HELD; ++j) raw[j] = i + 32 * j + lane < to ? ids[i + 32 * j + lane] : (Id)-1;
#pragma unroll
        for (int j = 0; j < RT_HELD; ++j) held[j] = raw[j] >= 0 && raw[j] < experts ? (int)raw[j] : (i + 32 * j + lane < to ? experts : -1);  // `experts`: of none
    };
    int mine = 0, less = 0;
    for (int i = from; i < to; i += CHUNK) {
        read(i);
#pragma unroll
        for (int j = 0; j < RT_HELD; ++j) {
            mine += held[j] == e;
            less += (unsigned)held[j] < (unsigned)e;  // (-1 is above)
        }
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    less = __reduce_add_sync(0xffffffffu, less);
    if (lane == 0) {
        before[warp] = mine;
        lower[warp] = less;
    }
    __syncthreads();
    // this warp's first row: the slots of lower experts, and those of this one in earlier pieces
    const int first = __reduce_add_sync(0xffffffffu, lower[lane]);
    int row = first + __reduce_add_sync(0xffffffffu, lane < warp ? before[lane] : 0);
    if (threadIdx.x == 0) offsets[e] = first;  // of e = experts: how many rows there are
    for (int i = from; i < to; i += CHUNK) {
        if (piece > CHUNK) read(i);
#pragma unroll
        for (int j = 0; j < RT_HELD; ++j) {
            const unsigned vote = __ballot_sync(0xffffffffu, held[j] == e);
            if (held[j] == e) {
                const int r = row + __popc(vote & ((1u << lane) - 1)), slot = i + 32 * j + lane;
                position[slot] = e < experts ? r : -1;
                order[r] = e < experts ? slot : -1;
            }
            row += __popc(vote);
        }
    }
}
static_assert(RT_THREADS == 1024, "a lane per warp adds up the warps' counts");

cudaError_t route_sort(const void* ids, bool wide, int slots, int experts, int* order, int* offsets, int* position, cudaStream_t s) {
    const dim3 grid((unsigned)experts + 1, 1, 1);
    if (wide) return launch_kernel(route_sort_kernel<long long>, grid, RT_THREADS, 0, s, false, static_cast<const long long*>(ids), slots, experts, order, offsets, position);
    return launch_kernel(route_sort_kernel<int>, grid, RT_THREADS, 0, s, false, static_cast<const int*>(ids), slots, experts, order, offsets, position);
}

// A thread's values of a row as they lie in memory. WIDE: V neighbouring ones from column c on, as many as fill the 16 bytes of a store
// (two half-filled stores per lane would leave every sector half written). Otherwise, for rows at any alignment, columns c, c + step, ...:
// a warp's loads are still neighbouring values, and V of them are under way per thread.
template <typename T, int V, bool WIDE> struct Values {
    alignas(WIDE ? (V * sizeof(T) >= 16 ? 16 : 8) : sizeof(T)) T raw[V];
    __device__ __forceinline__ void load(const T* row, int c, int step, int h) {
        if constexpr (!WIDE) {
#pragma unroll
            for (int i = 0; i < V; ++i) raw[i] = c + i * step < h ? row[c + i * step] : from_float<T>(0.0f);
        } else if constexpr (V * sizeof(T) == 8) {
            *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(row + c);
        } else {
#pragma unroll
            for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) reinterpret_cast<uint4*>(raw)[i] = *(reinterpret_cast<const uint4*>(row + c) + i);
        }
    }
    __device__ __forceinline__ void store(T* row, int c, int step, int h) const {
        if constexpr (!WIDE) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i * step < h) row[c + i * step] = raw[i];
        } else {  // (never less than 16 bytes)
#pragma unroll
            for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) reinterpret_cast<uint4*>(row + c)[i] = reinterpret_cast<const uint4*>(raw)[i];
        }
    }
    __device__ __forceinline__ float get(int i) const { return to_float<T>(raw[i]); }
    __device__ __forceinline__ void set(int i, float v) { raw[i] = from_float<T>(v); }
};
// the first column of a thread's loop over a row
template <int V, bool WIDE> __device__ __forceinline__ int first_column() { return WIDE ? V * threadIdx.x : threadIdx.x; }
static bool rows_wide(const void* p, long long ld, int elem) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (elem == ELEM_F32 ? 4 : 2) % 16 == 0;
}

// The rows of slots j.. of a token: -1 where there is none.
template <int S> __device__ __forceinline__ void slot_rows(const int* position, long long token, int topk, int j, int limit, int (&p)[S]) {
#pragma unroll
    for (int i = 0; i < S; ++i) p[i] = j + i < topk ? position[token * topk + j + i] : -1;
#pragma unroll
    for (int i = 0; i < S; ++i) p[i] = p[i] < limit ? p[i] : -1;
}

// A CTA per token reads it once and writes its rows; rows behind the last are zeroed by the CTA that they would have belonged to had no
// slot been left out.
template <typename U, int S>
__global__ void __launch_bounds__(RT_ROW_THREADS) route_dispatch_kernel(const U* __restrict__ x, long long ldx, const int* __restrict__ position,
                                                             const int* __restrict__ valid, U* __restrict__ rows, int topk, int h) {
    const long long t = blockIdx.x;
    const U* src = x + t * ldx;
    const int nvalid = min(*valid, (int)gridDim.x * topk);
    U zero{};
    for (int j = 0; j < topk; j += S) {
        int p[S];
        slot_rows(position, t, topk, j, nvalid, p);
        for (int c = (int)(blockIdx.y * blockDim.x + threadIdx.x); c < h; c += blockDim.x * gridDim.y) {
            const U v = src[c];
#pragma unroll
            for (int i = 0; i < S; ++i) {
                if (p[i] >= 0) rows[(long long)p[i] * h + c] = v;
                if (j + i < topk && t * topk + j + i >= nvalid) rows[(t * topk + j + i) * h + c] = zero;
            }
        }
    }
}

// threads of a CTA that goes over `n` pieces of a row
static unsigned row_threads(int n) { return n >= RT_ROW_THREADS ? (unsigned)RT_ROW_THREADS : (unsigned)((n + 31) / 32 * 32); }
// A CTA per token; where the tokens are too few to fill the SMs, more of them, each with its share of the columns (combine, f32, 8 slots,
// rows of 7168: 16 tokens 6.7 us with one CTA each, 2.6 with seven; 64 tokens 6.9 and 3.3).
static dim3 row_grid(int tokens, int n, unsigned threads) {
    const int steps = min((n + (int)threads - 1) / (int)threads, 256), room = runtime_info().sm_count * RT_ROW_CTAS / tokens;
    return dim3((unsigned)tokens, (unsigned)(room < 2 ? 1 : (steps < room ? steps : room)), 1);
}

cudaError_t route_dispatch(int elem, const void* x, long long ldx, const int* position, const int* valid, void* rows, int tokens, int topk, int h,
                           cudaStream_t s) {
    const int es = elem == ELEM_F32 ? 4 : 2;
    const auto go = [&](auto unit, int per) {  // `per` values in a unit
        using U = decltype(unit);
        const unsigned threads = row_threads(h / per);
        const auto kernel = topk <= 2 ? route_dispatch_kernel<U, 2> : route_dispatch_kernel<U, 4>;
        return launch_kernel(kernel, row_grid(tokens, h / per, threads), threads, 0, s, false, static_cast<const U*>(x), ldx / per, position, valid, static_cast<U*>(rows), topk, h / per);
    };
    if (rows_wide(x, ldx, elem) && rows_wide(rows, h, elem)) return go(uint4{}, 16 / es);
    if (es == 4) return go(uint32_t{}, 1);
    if (reinterpret_cast<uintptr_t>(x) % 4 == 0 && reinterpret_cast<uintptr_t>(rows) % 4 == 0 && ldx % 2 == 0 && h % 2 == 0) return go(uint32_t{}, 2);
    return go(uint16_t{}, 1);
}

// out[t] = sum_j weights[t, j] rows[position[t, j]]; weights null: 1. The loads of four slots' rows are under way at once: one after the
// other, eight slots of seven tokens took 7.4 us.
template <typename In, typename Out, int V, int S, bool WIDE>
__global__ void __launch_bounds__(RT_ROW_THREADS) route_combine_kernel(const In* rows, long long ldr, const int* position, const float* weights, Out* out, int topk,
                                                            int h) {
    grid_dependency_wait();
    grid_launch_dependents();
    const long long t = blockIdx.x;
    const int limit = (int)gridDim.x * topk;
    int p[S];
    float w[S];
    const auto slots = [&](int j) {
        slot_rows(position, t, topk, j, limit, p);
#pragma unroll
        for (int i = 0; i < S; ++i) w[i] = weights == nullptr ? 1.0f : (j + i < topk ? weights[t * topk + j + i] : 0.0f);
    };
    slots(0);
    for (int c = first_column<V, WIDE>() + (int)(blockIdx.y * V * blockDim.x); c < h; c += V * blockDim.x * gridDim.y) {
        float sum[V] = {};
        for (int j = 0; j < topk; j += S) {
            if (topk > S) slots(j);
            Values<In, V, WIDE> r[S];
#pragma unroll
            for (int i = 0; i < S; ++i)
                if (p[i] >= 0) r[i].load(rows + p[i] * ldr, c, blockDim.x, h);
#pragma unroll
            for (int i = 0; i < S; ++i)
                if (p[i] >= 0) {
#pragma unroll
                    for (int k = 0; k < V; ++k) sum[k] = fmaf(w[i], r[i].get(k), sum[k]);
                }
        }
        Values<Out, V, WIDE> v;
#pragma unroll
        for (int k = 0; k < V; ++k) v.set(k, sum[k]);
        v.store(out + t * h, c, blockDim.x, h);
    }
}

template <typename In, typename Out>
static cudaError_t combine_t(bool wide, const void* rows, long long ldr, const int* position, const float* weights, void* out, int tokens, int topk,
                             int h, cudaStream_t s, bool dependent) {
    constexpr int V = 16 / sizeof(Out);
    const int per = wide ? h / V : (h + 3) / 4;
    const unsigned threads = row_threads(per);
    const auto kernel = wide ? (topk <= 2 ? route_combine_kernel<In, Out, V, 2, true> : route_combine_kernel<In, Out, V, 4, true>) : route_combine_kernel<In, Out, 4, 4, false>;
    return launch_kernel(kernel, row_grid(tokens, per, threads), threads, 0, s, dependent, static_cast<const In*>(rows), ldr, position, weights, static_cast<Out*>(out), topk, h);
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

// The gradients of combine, a CTA per token: its slots' rows of drows (each written by one CTA), and the products with the rows, four
// slots at a time. Rows behind the last become zeros as in dispatch. Either output may be left out (null).
template <typename G, typename T, int V, int S, bool WIDE>
__global__ void __launch_bounds__(RT_ROW_THREADS) route_combine_grad_kernel(const G* __restrict__ grad_out, long long ldg, const T* __restrict__ rows, long long ldr,
                                                                 const int* __restrict__ position, const int* __restrict__ valid,
                                                                 const float* __restrict__ weights, T* __restrict__ grad_rows,
                                                                 float* __restrict__ grad_weights, int topk, int h) {
    __shared__ float part[S][RT_ROW_THREADS / 32];
    const long long t = blockIdx.x;
    const int nvalid = min(*valid, (int)gridDim.x * topk), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int j = 0; j < topk; j += S) {
        int p[S];
        slot_rows(position, t, topk, j, nvalid, p);
        float w[S], dot[S] = {};
#pragma unroll
        for (int i = 0; i < S; ++i) w[i] = j + i < topk ? weights[t * topk + j + i] : 0.0f;
        for (int c = first_column<V, WIDE>(); c < h; c += V * blockDim.x) {
            Values<G, V, WIDE> g;
            g.load(grad_out + t * ldg, c, blockDim.x, h);
            if (grad_weights != nullptr) {
                Values<T, V, WIDE> r[S];
#pragma unroll
                for (int i = 0; i < S; ++i)
                    if (p[i] >= 0) r[i].load(rows + p[i] * ldr, c, blockDim.x, h);
#pragma unroll
                for (int i = 0; i < S; ++i)
                    if (p[i] >= 0) {
#pragma unroll
                        for (int k = 0; k < V; ++k) dot[i] = fmaf(g.get(k), r[i].get(k), dot[i]);
                    }
            }
            if (grad_rows != nullptr) {
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    Values<T, V, WIDE> d;
                    if (p[i] >= 0) {
#pragma unroll
                        for (int k = 0; k < V; ++k) d.set(k, w[i] * g.get(k));
                        d.store(grad_rows + (long long)p[i] * h, c, blockDim.x, h);
                    }
                    if (j + i < topk && t * topk + j + i >= nvalid) {
#pragma unroll
                        for (int k = 0; k < V; ++k) d.set(k, 0.0f);
                        d.store(grad_rows + (t * topk + j + i) * h, c, blockDim.x, h);
                    }
                }
            }
        }
        if (grad_weights != nullptr) {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const float sum = warp_sum(dot[i]);
                if (lane == 0) part[i][warp] = sum;
            }
            __syncthreads();
            if (threadIdx.x < S && j + (int)threadIdx.x < topk) {
                float sum = 0.0f;
                for (int i = 0; i < (int)(blockDim.x >> 5); ++i) sum += part[threadIdx.x][i];
                grad_weights[t * topk + j + threadIdx.x] = sum;
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
    constexpr int V = 16 / sizeof(T);
    const auto kernel = wide ? (topk <= 2 ? route_combine_grad_kernel<G, T, V, 2, true> : route_combine_grad_kernel<G, T, V, 4, true>) : route_combine_grad_kernel<G, T, 4, 4, false>;
    return launch_kernel(kernel, grid, h >= 8 ? row_threads(wide ? h / V : (h + 3) / 4) : 32u, 0, s, false, g, ldg, r, ldr, position, valid, weights, d, grad_weights, topk, h);
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
