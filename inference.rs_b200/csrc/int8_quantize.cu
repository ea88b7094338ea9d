// Rows of f32 / f16 / bf16 -> int8 with one scale per row, and back.
//
//   s = max|x| / 127, rounded to 32 bits;   q = the integer next to x / s, ties to the even one.
//
// (Values so small that s is no normal float, under 1.5e-36, may have quotients above 127: they count as 127.)
//
// The quotient is never formed by division: t = x * (1 / s) is off by less than 2e-5, so round(t) is the integer unless t lies that
// close to a half, and there the remainder x - q s, which one fused multiply-add gives exactly (|q| <= 127 and s have 31 bits together,
// and the remainder is a multiple of half the last place of s), decides. A row with an infinity or a NaN in it has a NaN for a scale and
// zeros for integers: its products are NaN, as they would be in floating point, and no other row's.
//
// Bound by HBM: a row is read once, held in registers between the maximum and the rounding, and written as one byte a value.
#include "int8.cuh"

namespace b200q {

struct QuantizeRows {
    const void* x;
    long long ldx;
    int8_t* q;
    long long ldq;  // a multiple of 16: the bytes from k to the next multiple of 16 are written as zeros
    float* scales;
    long long rows;
    int k;
    const int* position;  // where a row's copies go: rows position[r * topk ...] of q, none for -1; null: row r
    int topk;
    const int* row_limit;  // rows from here on are left alone (null: none)
};

struct RowScale {
    float s;    // as stored
    float sn, inv, pre, near_half;  // x * pre / sn is the same quotient, with sn far from the smallest floats
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    RowScale r;
    const bool finite = amax_bits < 0x7f800000u;
    r.s = finite ? __uint_as_float(amax_bits) / 127.0f : __uint_as_float(0x7fc00000u);
    r.pre = r.s < 1e-30f ? 18446744073709551616.0f : 1.0f;  // 2^64
    r.sn = r.s * r.pre;
    r.inv = finite && r.s > 0.0f ? 1.0f / r.sn : 0.0f;
    r.near_half = 0.4999f * r.sn;
    return r;
}
__device__ __noinline__ float nearest_quotient(float x, float qf, float sn) {
    const float rem = fmaf(-qf, sn, x), half = 0.5f * sn;
    const bool odd = ((int)qf & 1) != 0;
    if (rem > half || (rem == half && odd)) return qf + 1.0f;
    if (rem < -half || (rem == -half && odd)) return qf - 1.0f;
    return qf;
}
__device__ __forceinline__ uint32_t quantize_one(float x, const RowScale& r) {
    if (r.inv == 0.0f) return 0u;  // a row of zeros, or with a value that is not finite
    const float xs = x * r.pre;
    float qf = fmaf(xs, r.inv, 12582912.0f) - 12582912.0f;
    if (fabsf(fmaf(-qf, r.sn, xs)) > r.near_half) qf = nearest_quotient(xs, qf, r.sn);
    if (r.pre != 1.0f) qf = fminf(fmaxf(qf, -127.0f), 127.0f);
    return (uint32_t)(int)qf & 0xffu;
}

// Eight values of a row as they lie in memory. Plain loads: what they read may be the work of the launch before, which this one waited
// for after it had started.
template <typename T> struct Eight;
template <> struct Eight<float> {
    float4 a, b;
    __device__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p);
        b = *(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template <typename T> struct Eight {
    uint4 a;
    __device__ void load(const T* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ void zero() { a = make_uint4(0u, 0u, 0u, 0u); }
    __device__ void get(float (&v)[8]) const {
        const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float<T>(e[i]);
    }
};

__device__ __forceinline__ uint32_t block_max(uint32_t v) {
    __shared__ uint32_t part[32];
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    const uint32_t w = (threadIdx.x & 31) < (blockDim.x >> 5) ? part[threadIdx.x & 31] : 0u;
    return __reduce_max_sync(0xffffffffu, w);
}

__device__ __forceinline__ void store_scale(const QuantizeRows& p, long long row, float s) {
    if (p.position == nullptr) {
        p.scales[row] = s;
    } else {
        for (int j = 0; j < p.topk; ++j) {
            const int to = p.position[row * p.topk + j];
            if (to >= 0) p.scales[to] = s;
        }
    }
}

// One CTA per row, eight values per thread and step.
template <typename T, int STEPS> __global__ void __launch_bounds__(1024) int8_quantize_kernel(const QuantizeRows p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const long long row = blockIdx.x;
    if (p.row_limit != nullptr && row >= *p.row_limit) return;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const int step = blockDim.x * 8, first = threadIdx.x * 8;
    Eight<T> held[STEPS];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        if (first + i * step < p.k) held[i].load(x + first + i * step);
        else held[i].zero();
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        float v[8];
        held[i].get(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
    }
    const RowScale r = row_scale(block_max(amax));
    if (threadIdx.x == 0) store_scale(p, row, r.s);
    const int kp = (p.k + 15) & ~15;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int c = first + i * step;
        if (c >= kp) break;
        float v[8];
        held[i].get(v);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j >> 2] |= quantize_one(v[j], r) << (8 * (j & 3));
        if (p.position == nullptr) {
            *reinterpret_cast<uint2*>(p.q + row * p.ldq + c) = make_uint2(w[0], w[1]);
        } else {
            for (int j = 0; j < p.topk; ++j) {
                const int to = p.position[row * p.topk + j];
                if (to >= 0) *reinterpret_cast<uint2*>(p.q + (long long)to * p.ldq + c) = make_uint2(w[0], w[1]);
            }
        }
    }
}

// Any width, any alignment of x: a value at a time, the row read twice.
template <typename T> __global__ void __launch_bounds__(256) int8_quantize_plain_kernel(const QuantizeRows p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const long long row = blockIdx.x;
    if (p.row_limit != nullptr && row >= *p.row_limit) return;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    uint32_t amax = 0;
    for (int c = threadIdx.x; c < p.k; c += 256) amax = max(amax, __float_as_uint(to_float<T>(x[c])) & 0x7fffffffu);
    const RowScale r = row_scale(block_max(amax));
    if (threadIdx.x == 0) store_scale(p, row, r.s);
    const int kp = (p.k + 15) & ~15;
    for (int c = 4 * threadIdx.x; c < kp; c += 1024) {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < p.k) w |= quantize_one(to_float<T>(x[c + j]), r) << (8 * j);
        if (p.position == nullptr) {
            *reinterpret_cast<uint32_t*>(p.q + row * p.ldq + c) = w;
        } else {
            for (int j = 0; j < p.topk; ++j) {
                const int to = p.position[row * p.topk + j];
                if (to >= 0) *reinterpret_cast<uint32_t*>(p.q + (long long)to * p.ldq + c) = w;
            }
        }
    }
}

template <typename T> static cudaError_t quantize_t(const QuantizeRows& p, cudaStream_t s, bool dependent) {
    const bool wide = p.k % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.ldx * sizeof(T) % 16 == 0 && p.k <= 32768;
    const dim3 grid((unsigned)p.rows, 1, 1);
    if (!wide) return launch_kernel(int8_quantize_plain_kernel<T>, grid, 256, 0, s, dependent, p);
    const int eights = (p.k + 15) / 16 * 2, whole = (eights + 31) / 32 * 32;
    // few rows: every thread one step, the shortest way; many: four steps, so that more loads are under way per thread
    if (whole <= 1024 && (p.rows < 512 || whole <= 128)) return launch_kernel(int8_quantize_kernel<T, 1>, grid, (unsigned)whole, 0, s, dependent, p);
    return launch_kernel(int8_quantize_kernel<T, 4>, grid, (unsigned)((eights + 127) / 128 * 32), 0, s, dependent, p);
}

cudaError_t int8_quantize_rows(int elem, const void* x, long long ldx, int8_t* q, long long ldq, float* scales, long long rows, int k,
                               const int* position, int topk, const int* row_limit, cudaStream_t s, bool dependent) {
    const QuantizeRows p{x, ldx, q, ldq, scales, rows, k, position, topk, row_limit};
    if (elem == ELEM_F32) return quantize_t<float>(p, s, dependent);
    if (elem == ELEM_F16) return quantize_t<__half>(p, s, dependent);
    return quantize_t<__nv_bfloat16>(p, s, dependent);
}

template <typename T> __global__ void __launch_bounds__(256) int8_dequantize_kernel(const int8_t* __restrict__ q, long long ldq, const float* __restrict__ scales,
                                                                                    T* __restrict__ out, int k, int wide) {
    const long long row = blockIdx.x;
    const float s = scales[row];
    const int8_t* src = q + row * ldq;
    T* dst = out + row * k;
    if (wide) {
        for (int c = 8 * threadIdx.x; c < k; c += 2048) {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(src + c));
            alignas(16) T v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = from_float<T>((float)(int8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3))) * s);
#pragma unroll
            for (int j = 0; j < (int)(sizeof(v) / 16); ++j) reinterpret_cast<uint4*>(dst + c)[j] = reinterpret_cast<const uint4*>(v)[j];
        }
    } else {
        for (int c = threadIdx.x; c < k; c += 256) dst[c] = from_float<T>((float)src[c] * s);
    }
}

cudaError_t int8_dequantize_rows(int elem, const int8_t* q, long long ldq, const float* scales, void* out, long long rows, int k, cudaStream_t s) {
    const int wide = k % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    const dim3 grid((unsigned)rows, 1, 1);
    if (elem == ELEM_F32) return launch_kernel(int8_dequantize_kernel<float>, grid, 256, 0, s, false, q, ldq, scales, static_cast<float*>(out), k, wide);
    if (elem == ELEM_F16) return launch_kernel(int8_dequantize_kernel<__half>, grid, 256, 0, s, false, q, ldq, scales, static_cast<__half*>(out), k, wide);
    return launch_kernel(int8_dequantize_kernel<__nv_bfloat16>, grid, 256, 0, s, false, q, ldq, scales, static_cast<__nv_bfloat16*>(out), k, wide);
}

}  // namespace b200q
