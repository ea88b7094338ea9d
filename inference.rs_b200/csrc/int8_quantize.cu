// Rows of f32 / f16 / bf16 -> int8 with one scale per row, and back.
//
//   s = max|x| / 127, rounded to 32 bits;   q = the integer next to x / s, ties to the even one.
//
// (Values so small that s is no normal float, under 1.5e-36, may have quotients above 127: they count as 127.)
//
// The quotient is never formed by division: t = x * (1 / s) is off by less than 2e-5, so round(t) is the integer unless t lies that
// close to a half, and there the remainder x - q s, which one fused multiply-add gives exactly (it is a multiple of half the last place
// of s, and not much more than s / 2), decides. A row with an infinity or a NaN in it has a NaN for a scale and
// zeros for integers: its products are NaN, as they would be in floating point, and no other row's.
//
// Bound by HBM: a row is read once, held in registers between the maximum and the rounding, and written as one byte a value.
#include <type_traits>

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
    // routing in the same launch (int8_route_quantize): the slots' expert ids, and what route_sort would make of them
    const void* ids;
    bool wide_ids;
    int experts;
    int *position_out, *offsets;
};

constexpr float ROUND = 12582912.0f;  // 1.5 * 2^23: v + ROUND has the integer next to v in its low bits

struct RowScale {
    float s;          // as stored
    float sn, inv;    // x * pre / sn is the same quotient, with sn far from the smallest floats; inv 0: the integers are zeros
    float pre, half;  // half of sn
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    RowScale r;
    const bool finite = amax_bits < 0x7f800000u;
    r.s = finite ? __uint_as_float(amax_bits) / 127.0f : __uint_as_float(0x7fc00000u);
    r.pre = r.s < 1e-30f ? 18446744073709551616.0f : 1.0f;  // 2^64
    r.sn = r.s * r.pre;
    r.inv = finite && r.s > 0.0f ? 1.0f / r.sn : 0.0f;
    r.half = 0.5f * r.sn;
    return r;
}
// Four values, one byte each, where a value may lie exactly on a half, or the scale is among the smallest floats.
__device__ __noinline__ uint32_t quantize_four_carefully(float a, float b, float c, float d, float sn, float inv, float pre) {
    const float v[4] = {a, b, c, d}, half = 0.5f * sn;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = v[i] * pre;
        float q = fmaf(x, inv, ROUND) - ROUND;
        const float rem = fmaf(-q, sn, x);
        const bool odd = ((int)q & 1) != 0;
        if (rem > half || (rem == half && odd)) q += 1.0f;
        else if (rem < -half || (rem == -half && odd)) q -= 1.0f;
        w |= ((uint32_t)(int)fminf(fmaxf(q, -127.0f), 127.0f) & 0xffu) << (8 * i);
    }
    return w;
}
// The remainder settles every value without a branch: one bf16 value in some hundred has a quotient within a rounding of s of a half (127
// times one 8-bit mantissa by another), so a way out of line for them was taken by every other warp and cost as much as all the rest.
// A value can lie on a half exactly without s being a power of two, for which the rounding of x * (1 / s) is right as it is. Not so for
// bf16: half an odd multiple of s has 8 bits only where s has one. In an f16 row in a hundred s has few bits and many values lie there: they
// are settled in line (512 rows of 4096: by a way out of line 5.8 us, now 3.6). f32 values hardly ever do, and the way out of line is the
// faster one (8192 rows of 14336: 101 us, in line 108.6).
// Rows of the smallest floats (r.pre) are not for this one.
template <typename T> __device__ __forceinline__ uint32_t quantize_four(float a, float b, float c, float d, const RowScale& r) {
    const float v[4] = {a, b, c, d};
    float t[4];
    bool on_half = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        t[i] = fmaf(v[i], r.inv, ROUND);
        const float rem = fmaf(ROUND - t[i], r.sn, v[i]);
        if constexpr (sizeof(T) == 4) on_half |= fabsf(rem) == r.half;
        const float step = __uint_as_float((__float_as_uint(rem) & 0x80000000u) | 0x3f800000u);
        uint32_t size = __float_as_uint(rem) & 0x7fffffffu;
        // an odd integer gives way to the even one next to it, as if its remainder were larger by the last place
        if constexpr (std::is_same<T, __half>::value) size += __float_as_uint(t[i]) & 1u;
        t[i] = __uint_as_float(size) > r.half ? t[i] + step : t[i];
    }
    if (sizeof(T) == 4 && on_half) return quantize_four_carefully(a, b, c, d, r.sn, r.inv, 1.0f);
    return __byte_perm(__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040), __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
}

template <typename T> __device__ __forceinline__ uint32_t quantize_any(float a, float b, float c, float d, const RowScale& r) {
    if (r.inv == 0.0f) return 0u;
    return r.pre == 1.0f ? quantize_four<T>(a, b, c, d, r) : quantize_four_carefully(a, b, c, d, r.sn, r.inv, r.pre);
}

// Eight values of a row as they lie in memory. Plain loads: what they read may be the work of the launch before, which this one waited
// for after it had started. `top` is the largest magnitude, `float_bits` its pattern as a float: patterns without their sign are in the
// order of the values, with infinities and NaN above all.
template <typename T> struct Eight;
template <> struct Eight<float> {
    float4 a, b;
    __device__ void load(const float* p) {
        a = *reinterpret_cast<const float4*>(p);
        b = *(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ void load_some(const float* x, int c, int k) {  // of x[c..c + 8) what lies in [0, k)
        float* v[8] = {&a.x, &a.y, &a.z, &a.w, &b.x, &b.y, &b.z, &b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i >= 0 && c + i < k) *v[i] = x[c + i];
    }
    static __device__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
    __device__ uint32_t top(uint32_t m) const {
        m = max(m, max(max(abs_bits(a.x), abs_bits(a.y)), max(abs_bits(a.z), abs_bits(a.w))));
        return max(m, max(max(abs_bits(b.x), abs_bits(b.y)), max(abs_bits(b.z), abs_bits(b.w))));
    }
    static __device__ uint32_t float_bits(uint32_t top) { return top; }
    __device__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template <typename T> struct Eight {
    uint4 a;
    __device__ void load(const T* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ void zero() { a = make_uint4(0u, 0u, 0u, 0u); }
    __device__ void load_some(const T* x, int c, int k) {
        uint32_t* w[4] = {&a.x, &a.y, &a.z, &a.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i >= 0 && c + i < k) *w[i / 2] |= (uint32_t)*reinterpret_cast<const unsigned short*>(x + c + i) << (16 * (i & 1));
    }
    using Pair = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    __device__ uint32_t top(uint32_t m) const {  // two values side by side, a NaN above all
        const Pair* w = reinterpret_cast<const Pair*>(&a);
        const Pair lo = __hmax2_nan(__habs2(w[0]), __habs2(w[1])), hi = __hmax2_nan(__habs2(w[2]), __habs2(w[3]));
        const Pair r = __hmax2_nan(*reinterpret_cast<const Pair*>(&m), __hmax2_nan(lo, hi));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ uint32_t float_bits(uint32_t top) {
        const unsigned short lo = (unsigned short)top, hi = (unsigned short)(top >> 16);
        return max(__float_as_uint(to_float<T>(*reinterpret_cast<const T*>(&lo))) & 0x7fffffffu, __float_as_uint(to_float<T>(*reinterpret_cast<const T*>(&hi))) & 0x7fffffffu);
    }
    __device__ void get(float (&v)[8]) const {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
            const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_float<T>(e[i]);
        }
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

// The rows of q that a row goes to: itself (to null), or those of `to` that are there.
template <typename Fn> __device__ __forceinline__ void each_target(const QuantizeRows& p, long long row, const int* to, Fn fn) {
    if (to == nullptr) {
        fn(row);
    } else {
        for (int j = 0; j < p.topk; ++j)
            if (to[j] >= 0) fn((long long)to[j]);
    }
}
__device__ __forceinline__ const int* targets(const QuantizeRows& p, long long row) { return p.position != nullptr ? p.position + row * p.topk : nullptr; }

// `size` threads (a warp or a CTA) and their share of a row: eight values per thread and step, group g of them with rank g % size.
// ODD: a row starts anywhere. Its groups are those between 16-byte boundaries, so that the first holds `head` values of what lies before
// (and counts them as zeros, as the last does with what lies behind; these two are read value by value), and a group's integers are
// those of two neighbours, `head` bytes on.
template <typename T, int STEPS, bool ODD> struct RowPart {
    Eight<T> held[STEPS];
    int head;
    __device__ __forceinline__ void load(const QuantizeRows& p, long long row, int rank, int size) {
        const T* x = static_cast<const T*>(p.x) + row * p.ldx;
        head = ODD ? (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T)) : 0;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int c = 8 * (rank + i * size) - head;
            if (c >= 0 && c + 8 <= p.k) {
                held[i].load(x + c);
            } else {
                held[i].zero();
                if constexpr (ODD) {
                    if (c < p.k) held[i].load_some(x, c, p.k);
                }
            }
        }
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) m = held[i].top(m);
        return Eight<T>::float_bits(m);
    }
    // by all of the threads; `next`: of the eight integers of a group and step, those of the group behind it
    template <typename Next> __device__ __forceinline__ void store(const QuantizeRows& p, long long row, const RowScale& r, int rank, int size, const int* to, Next next) const {
        const int kp = (p.k + 15) & ~15;
        if (rank == 0) each_target(p, row, to, [&](long long at) { p.scales[at] = r.s; });
        uint2 w[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            float v[8];
            held[i].get(v);
            w[i] = make_uint2(quantize_any<T>(v[0], v[1], v[2], v[3], r), quantize_any<T>(v[4], v[5], v[6], v[7], r));
        }
        if constexpr (ODD) next(w, head);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int c = 8 * (rank + i * size);
            if (c >= kp) break;
            each_target(p, row, to, [&](long long at) { *reinterpret_cast<uint2*>(p.q + at * p.ldq + c) = w[i]; });
        }
    }
};
// bytes `head`.. of two groups' sixteen
__device__ __forceinline__ uint2 shifted(uint2 a, uint2 b, int head) {
    const bool far = head >= 4;
    const uint32_t w0 = far ? a.y : a.x, w1 = far ? b.x : a.y, w2 = far ? b.y : b.x;
    return make_uint2(__funnelshift_r(w0, w1, 8 * (head & 3)), __funnelshift_r(w1, w2, 8 * (head & 3)));
}
__device__ __forceinline__ long long row_count(const QuantizeRows& p) {
    return p.row_limit != nullptr ? min((long long)max(*p.row_limit, 0), p.rows) : p.rows;
}

// Routing for few slots, without a launch of its own: the CTA of a token counts through all ids where its own slots go, and one more CTA
// finds where the experts' rows begin. What route_sort_kernel would give, in the same order.
constexpr int ROUTE_MOST_SLOTS = 2048, ROUTE_MOST_TOPK = 8;
__device__ __forceinline__ int expert_id(const QuantizeRows& p, int slot) { return expert_id(p.ids, p.wide_ids, p.experts, slot); }
__device__ __forceinline__ void route_token(const QuantizeRows& p, int token, int (&to)[ROUTE_MOST_TOPK]) {
    const int slots = (int)p.rows * p.topk, first = token * p.topk;
    int mine[ROUTE_MOST_TOPK], before[ROUTE_MOST_TOPK] = {};
#pragma unroll
    for (int j = 0; j < ROUTE_MOST_TOPK; ++j) mine[j] = j < p.topk ? expert_id(p, first + j) : -1;
    if (threadIdx.x < ROUTE_MOST_TOPK) to[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < slots; i += blockDim.x) {
        const int id = expert_id(p, i);
#pragma unroll
        for (int j = 0; j < ROUTE_MOST_TOPK; ++j) before[j] += id < mine[j] || (id == mine[j] && i < first + j);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ROUTE_MOST_TOPK; ++j) {
        if (j >= p.topk) break;
        const int sum = __reduce_add_sync(0xffffffffu, before[j]);
        if ((threadIdx.x & 31) == 0 && sum != 0) atomicAdd(&to[j], sum);  // (integers: any order)
    }
    __syncthreads();
    if ((int)threadIdx.x < p.topk) {
        if (expert_id(p, first + threadIdx.x) == p.experts) to[threadIdx.x] = -1;
        p.position_out[first + threadIdx.x] = to[threadIdx.x];
    }
    __syncthreads();
}
// A CTA per row; ODD rows pass their integers on through shared memory. ROUTE: see above.
template <typename T, int STEPS, int MAX_THREADS, bool ODD, bool ROUTE> __global__ void __launch_bounds__(MAX_THREADS) int8_quantize_kernel(const QuantizeRows p) {
    extern __shared__ uint2 groups[];
    __shared__ int to[ROUTE ? ROUTE_MOST_TOPK : 1];
    grid_dependency_wait();
    grid_launch_dependents();
    const long long row = blockIdx.x;
    if constexpr (ROUTE) {
        __shared__ int off[INT8_MAX_EXPERTS + 1];
        if (row == p.rows) {
            expert_offsets(p.ids, p.wide_ids, p.experts, (int)p.rows * p.topk, off);
            for (int e = threadIdx.x; e <= p.experts; e += blockDim.x) p.offsets[e] = off[e];
            return;
        }
    } else {
        if (row >= row_count(p)) return;
    }
    const int rank = threadIdx.x, size = blockDim.x;
    RowPart<T, STEPS, ODD> part;
    part.load(p, row, rank, size);
    if constexpr (ROUTE) route_token(p, (int)row, to);
    part.store(p, row, row_scale(block_max(part.top())), rank, size, ROUTE ? to : targets(p, row), [&](uint2 (&w)[STEPS], int head) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) groups[rank + i * size] = w[i];
        if (rank == 0) groups[STEPS * size] = make_uint2(0u, 0u);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < STEPS; ++i) w[i] = shifted(w[i], groups[rank + i * size + 1], head);
    });
}
// A warp per row, rows of up to 1024 values, of up to 1536 where there are many: a CTA for each such row would cost its start, about a
// nanosecond (bf16 of 1408: 24576 rows 28.9 us by CTAs, 21.5 by warps; 1024 rows 3.3 and 3.1, 512 2.9 and 3.1; of 2048, 24576 rows, 29.3
// and 27.1, f32 38.8 and 39.6).
constexpr int SHORT_ROWS = 1024;
template <typename T, int STEPS, bool ODD> __global__ void __launch_bounds__(256) int8_quantize_short_kernel(const QuantizeRows p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= row_count(p)) return;
    RowPart<T, STEPS, ODD> part;
    part.load(p, row, lane, 32);
    part.store(p, row, row_scale(__reduce_max_sync(0xffffffffu, part.top())), lane, 32, targets(p, row), [&](uint2 (&w)[STEPS], int head) {
        uint2 behind[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const uint2 first = i < STEPS - 1 ? w[i + 1] : make_uint2(0u, 0u);  // lane 31's neighbour: lane 0 of the next step
            behind[i] = make_uint2(__shfl_down_sync(0xffffffffu, w[i].x, 1), __shfl_down_sync(0xffffffffu, w[i].y, 1));
            const uint2 wrap = make_uint2(__shfl_sync(0xffffffffu, first.x, 0), __shfl_sync(0xffffffffu, first.y, 0));
            if (lane == 31) behind[i] = wrap;
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i) w[i] = shifted(w[i], behind[i], head);
    });
}

// Rows too wide to hold: a value at a time, the row read twice.
template <typename T> __global__ void __launch_bounds__(256) int8_quantize_plain_kernel(const QuantizeRows p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const long long row = blockIdx.x;
    if (p.row_limit != nullptr && row >= *p.row_limit) return;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    uint32_t amax = 0;
    for (int c = threadIdx.x; c < p.k; c += 256) amax = max(amax, __float_as_uint(to_float<T>(x[c])) & 0x7fffffffu);
    const RowScale r = row_scale(block_max(amax));
    const int* to = targets(p, row);
    if (threadIdx.x == 0) each_target(p, row, to, [&](long long at) { p.scales[at] = r.s; });
    const int kp = (p.k + 15) & ~15;
    for (int c = 4 * threadIdx.x; c < kp; c += 1024) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c + j < p.k ? to_float<T>(x[c + j]) : 0.0f;
        const uint32_t w = quantize_any<T>(v[0], v[1], v[2], v[3], r);
        each_target(p, row, to, [&](long long at) { *reinterpret_cast<uint32_t*>(p.q + at * p.ldq + c) = w; });
    }
}

template <typename T, bool ODD> static cudaError_t quantize_held(const QuantizeRows& p, cudaStream_t s, bool dependent) {
    if (p.k > (ODD ? 32768 - 16 : 32768)) return launch_kernel(int8_quantize_plain_kernel<T>, dim3((unsigned)p.rows, 1, 1), 256, 0, s, dependent, p);
    const long long sms = runtime_info().sm_count;
    const int eights = (p.k + 15) / 16 * 2 + (ODD ? 1 : 0), whole = (eights + 31) / 32 * 32;
    const auto go = [&](auto kernel, unsigned threads, int steps) {
        return launch_kernel(kernel, dim3((unsigned)p.rows, 1, 1), threads, ODD ? (threads * steps + 1) * sizeof(uint2) : 0, s, dependent, p);
    };
    // few rows: every thread as few steps as there can be, the shortest way
    if (p.rows <= 2 * sms && whole <= 1024) return go(int8_quantize_kernel<T, 1, 1024, ODD, false>, (unsigned)whole, 1);
    if (eights <= 128 || (eights <= 192 && p.rows >= SHORT_ROWS)) {
        const auto kernel = eights <= 32 ? int8_quantize_short_kernel<T, 1, ODD> : eights <= 64 ? int8_quantize_short_kernel<T, 2, ODD>
                          : eights <= 128 ? int8_quantize_short_kernel<T, 4, ODD> : int8_quantize_short_kernel<T, 6, ODD>;
        return launch_kernel(kernel, dim3((unsigned)((p.rows + 7) / 8), 1, 1), 256, 0, s, dependent, p);
    }
    const unsigned threads = (unsigned)((eights + 127) / 128 * 32);
    if (threads <= 512) return go(int8_quantize_kernel<T, 4, 512, ODD, false>, threads, 4);
    return go(int8_quantize_kernel<T, 4, 1024, ODD, false>, threads, 4);
}
template <typename T> static bool starts_anywhere(const QuantizeRows& p) {
    return p.k % 8 != 0 || reinterpret_cast<uintptr_t>(p.x) % 16 != 0 || p.ldx * sizeof(T) % 16 != 0;
}
template <typename T, bool ODD> static cudaError_t route_held(const QuantizeRows& p, cudaStream_t s) {
    const unsigned threads = (unsigned)(((p.k + 15) / 16 * 2 + (ODD ? 1 : 0) + 31) / 32 * 32);
    return launch_kernel(int8_quantize_kernel<T, 1, 1024, ODD, true>, dim3((unsigned)p.rows + 1, 1, 1), threads, ODD ? (threads + 1) * sizeof(uint2) : 0, s, false, p);
}
template <typename T> static cudaError_t route_t(const QuantizeRows& p, cudaStream_t s) { return starts_anywhere<T>(p) ? route_held<T, true>(p, s) : route_held<T, false>(p, s); }

// One launch (2 us) less for the layer of experts where every CTA can look at all ids and hold a row.
bool int8_routes_quantizing(int tokens, int topk, int k) {
    return topk <= ROUTE_MOST_TOPK && tokens * topk <= ROUTE_MOST_SLOTS && tokens <= 2 * runtime_info().sm_count && k <= 8192 - 16;
}
cudaError_t int8_route_quantize(int elem, const void* x, long long ldx, int8_t* q, long long ldq, float* scales, int tokens, int k, const void* ids,
                                bool wide_ids, int topk, int experts, int* position, int* offsets, cudaStream_t s) {
    const QuantizeRows p{x, ldx, q, ldq, scales, tokens, k, nullptr, topk, nullptr, ids, wide_ids, experts, position, offsets};
    if (elem == ELEM_F32) return route_t<float>(p, s);
    if (elem == ELEM_F16) return route_t<__half>(p, s);
    return route_t<__nv_bfloat16>(p, s);
}

template <typename T> static cudaError_t quantize_t(const QuantizeRows& p, cudaStream_t s, bool dependent) {
    const bool odd = starts_anywhere<T>(p);
    return odd ? quantize_held<T, true>(p, s, dependent) : quantize_held<T, false>(p, s, dependent);
}

cudaError_t int8_quantize_rows(int elem, const void* x, long long ldx, int8_t* q, long long ldq, float* scales, long long rows, int k,
                               const int* position, int topk, const int* row_limit, cudaStream_t s, bool dependent) {
    const QuantizeRows p{x, ldx, q, ldq, scales, rows, k, position, topk, row_limit, nullptr, false, 0, nullptr, nullptr};
    if (elem == ELEM_F32) return quantize_t<float>(p, s, dependent);
    if (elem == ELEM_F16) return quantize_t<__half>(p, s, dependent);
    return quantize_t<__nv_bfloat16>(p, s, dependent);
}

// 16 bytes of values per thread and step, one store: a row's groups are those between 16-byte boundaries of the output, and their integers
// are shifted out of aligned words. ODD: rows start anywhere, and their first and last groups are written value by value. SIZE threads
// per row, so that short rows share a CTA. (Two stores side by side per lane, which leave every sector half written: f32, 14336 x 4096,
// 55 us against 46.)
template <typename T, int SIZE, bool ODD> __global__ void __launch_bounds__(256) int8_dequantize_kernel(const int8_t* __restrict__ q, long long ldq, const float* __restrict__ scales,
                                                                                              T* __restrict__ out, long long rows, int k) {
    constexpr int V = 16 / sizeof(T);
    const long long row = (long long)blockIdx.x * (256 / SIZE) + threadIdx.x / SIZE;
    if (row >= rows) return;
    const float s = scales[row];
    const int8_t* src = q + row * ldq;
    T* dst = out + row * k;
    const int head = ODD ? (int)(reinterpret_cast<uintptr_t>(dst) % 16 / sizeof(T)) : 0, shift = 8 * (-head & 3);
#pragma unroll 4
    for (int c = V * (int)(threadIdx.x % SIZE) - head; c < k; c += V * SIZE) {
        if (!ODD || (c >= 0 && c + V <= k)) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(src + (c & ~3));
            uint32_t b[V / 4 + 1];
#pragma unroll
            for (int j = 0; j < V / 4; ++j) b[j] = __ldg(w + j);
            b[V / 4] = ODD && shift != 0 ? __ldg(w + V / 4) : 0u;
            alignas(16) T v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = from_float<T>((float)(int8_t)(__funnelshift_r(b[j / 4], b[j / 4 + 1], shift) >> (8 * (j % 4))) * s);
            *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(v);
        } else {
            for (int j = max(0, -c); j < min(V, k - c); ++j) dst[c + j] = from_float<T>((float)src[c + j] * s);
        }
    }
}
template <typename T> static cudaError_t dequantize_t(const int8_t* q, long long ldq, const float* scales, void* out, long long rows, int k, cudaStream_t s) {
    const bool shared = k <= 1024, odd = reinterpret_cast<uintptr_t>(out) % 16 != 0 || k % (16 / sizeof(T)) != 0;
    const auto kernel = odd ? (shared ? int8_dequantize_kernel<T, 32, true> : int8_dequantize_kernel<T, 256, true>)
                            : (shared ? int8_dequantize_kernel<T, 32, false> : int8_dequantize_kernel<T, 256, false>);
    return launch_kernel(kernel, dim3((unsigned)(shared ? (rows + 7) / 8 : rows), 1, 1), 256, 0, s, false, q, ldq, scales, static_cast<T*>(out), rows, k);
}

cudaError_t int8_dequantize_rows(int elem, const int8_t* q, long long ldq, const float* scales, void* out, long long rows, int k, cudaStream_t s) {
    if (elem == ELEM_F32) return dequantize_t<float>(q, ldq, scales, out, rows, k, s);
    if (elem == ELEM_F16) return dequantize_t<__half>(q, ldq, scales, out, rows, k, s);
    return dequantize_t<__nv_bfloat16>(q, ldq, scales, out, rows, k, s);
}

}  // namespace b200q
