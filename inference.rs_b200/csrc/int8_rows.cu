// Products of int8 rows on warp-level integer MMAs: a CTA owns 16 or 32 weight rows of one matrix and reads them once for up to 32
// tokens, straight from global memory into MMA fragments. The warps of a CTA share the k range and add up through shared memory;
// the sums are integers, so their order changes nothing.
//
// A lane loads 16 neighbouring bytes of a row: of the four words two make its part of one 32-k MMA and two that of the next. That takes
// the k of a 64-byte piece in another order than they lie, the same one for weights and tokens, which a sum does not mind.
#include "int8.cuh"

namespace b200q {

constexpr int I8R_WARPS = 8;
constexpr int I8R_STEP = 64;  // k of one piece

__device__ __forceinline__ uint4 ldg_stream(const int8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename OutT, int R, int NT>
__global__ void __launch_bounds__(32 * I8R_WARPS) int8_rows_kernel(const Int8Product p) {
    constexpr int ROWS = 16 * R, TOKENS = 8 * NT, PITCH = ROWS + 4;
    __shared__ int sums[I8R_WARPS][TOKENS][PITCH];
    grid_dependency_wait();
    grid_launch_dependents();
    const int e = blockIdx.y, row0 = blockIdx.x * ROWS;
    const int first = p.offsets != nullptr ? max(p.offsets[e], 0) : 0, last = p.offsets != nullptr ? min(p.offsets[e + 1], p.rows) : p.rows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int8_t* w[2 * R];
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) w[i] = p.wq + ((long long)e * p.n + min(row0 + 8 * i + g, p.n - 1)) * p.ldw + 16 * t;
    const int kp = (p.k + 15) & ~15, steps = (kp + I8R_STEP - 1) / I8R_STEP;
    for (int tok0 = first; tok0 < last; tok0 += TOKENS) {
        const int8_t* x[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) x[j] = p.xq + (long long)min(tok0 + 8 * j + g, last - 1) * p.ldx + 16 * t;
        int acc[R][NT][4] = {};
#pragma unroll 2
        for (int s = warp; s < steps; s += I8R_WARPS) {
            const int k0 = s * I8R_STEP;
            const bool in = k0 + 16 * t < kp;
            uint4 a[2 * R], b[NT];
#pragma unroll
            for (int i = 0; i < 2 * R; ++i) a[i] = in ? ldg_stream(w[i] + k0) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j] = in ? *reinterpret_cast<const uint4*>(x[j] + k0) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    mma_s8(acc[i][j], a[2 * i].x, a[2 * i + 1].x, a[2 * i].y, a[2 * i + 1].y, b[j].x, b[j].y);
                    mma_s8(acc[i][j], a[2 * i].z, a[2 * i + 1].z, a[2 * i].w, a[2 * i + 1].w, b[j].z, b[j].w);
                }
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) sums[warp][8 * j + 2 * t + (c & 1)][16 * i + g + 8 * (c >> 1)] = acc[i][j][c];
        __syncthreads();
        const int toks = min(TOKENS, last - tok0);
        auto value = [&](int tok, int r) {
            int sum = 0;
#pragma unroll
            for (int v = 0; v < I8R_WARPS; ++v) sum += sums[v][tok][r];
            return (float)sum * p.xs[tok0 + tok] * p.ws[(long long)e * p.n + row0 + r];
        };
        OutT* y = static_cast<OutT*>(p.y) + (long long)tok0 * p.ldy;
        if (p.act == INT8_ACT_NONE) {
            for (int i = threadIdx.x; i < toks * ROWS; i += 32 * I8R_WARPS) {
                const int r = i % ROWS, tok = i / ROWS;
                if (row0 + r < p.n) y[tok * p.ldy + row0 + r] = from_float<OutT>(value(tok, r));
            }
        } else {
            for (int i = threadIdx.x; i < toks * ROWS / 2; i += 32 * I8R_WARPS) {
                const int c = i % (ROWS / 2), tok = i / (ROWS / 2), r = (c & ~7) * 2 + (c & 7);
                if (row0 / 2 + c < p.n_out) y[tok * p.ldy + row0 / 2 + c] = from_float<OutT>(int8_activate(value(tok, r), p.act) * value(tok, r + 8));
            }
        }
        __syncthreads();
    }
}

template <typename OutT> static cudaError_t rows_t(const Int8Product& p, cudaStream_t s, bool dependent) {
    const int per = p.experts > 1 ? (p.rows + p.experts - 1) / p.experts : p.rows;  // tokens of an expert, on average
    const int r16 = (p.n + 15) / 16, r32 = (p.n + 31) / 32;
    if (per <= 8) return launch_kernel(int8_rows_kernel<OutT, 1, 1>, dim3(r16, p.experts), 32 * I8R_WARPS, 0, s, dependent, p);
    if (per <= 16) return launch_kernel(int8_rows_kernel<OutT, 1, 2>, dim3(r16, p.experts), 32 * I8R_WARPS, 0, s, dependent, p);
    return launch_kernel(int8_rows_kernel<OutT, 2, 4>, dim3(r32, p.experts), 32 * I8R_WARPS, 0, s, dependent, p);
}

cudaError_t int8_product_rows(int elem, const Int8Product& p, cudaStream_t s, bool dependent) {
    if (elem == ELEM_F32) return rows_t<float>(p, s, dependent);
    if (elem == ELEM_F16) return rows_t<__half>(p, s, dependent);
    return rows_t<__nv_bfloat16>(p, s, dependent);
}

}  // namespace b200q
