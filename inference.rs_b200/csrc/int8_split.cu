// The product of int8_pair.cu for few tiles: with 16 tiles of 256 rows and 74 pairs of SMs, two or four pairs take a tile, each a part of
// k, and add up through each other's shared memory. A cluster of 4 or 8 CTAs holds the pairs of a tile; when their products are done,
// each sends the sums of a part of the tokens to the pair that finishes them. Integers: the order of the sums does not matter.
//
// Without it 64 tokens of 14336 x 4096 run on 32 SMs, each fetching operands as fast as one SM can. us, quantizer included, undivided ->
// divided: 64 x 14336 x 4096 23.5 -> 17.6 (HBM needs 9.3), 256 x 14336 x 1024 28.3 -> 16.2, 256 x 14336 x 4096 30.6 -> 22.8, 256 x 4096 x
// 4096 13.6 -> 12.5, 128 x 2048 x 2048 9.8 -> 9.3. Tiles of up to 128 tokens: higher ones have more sums to send than their products save
// (256 x 4096 x 4096 in tiles of 256 15.3). Parts through global memory instead, by whichever pair comes last, cost 4 us more.
//
// Every wait is bounded, as in int8_pair.cu; a CTA that gave up still comes to the cluster's barriers.
#include <atomic>

#include "int8_pair.cuh"

namespace b200q {

constexpr int I8S_TOKENS = 128;  // of a tile at most = TMEM columns
constexpr int I8S_LEAST = 16;  // pieces of 128 k that are worth dividing
constexpr int I8S_CHUNK = 32 * I8P_ROWS;  // sums of 32 tokens of a CTA's rows

struct Int8SplitParams {
    Int8Product p;
    int bn, stages, tiles_m;
};
struct Int8SplitBarriers {
    uint64_t full[I8P_MAX_STAGES], empty[I8P_MAX_STAGES], done;
    uint32_t tmem_base;
};
static size_t i8s_smem(int stages, int bn) { return 1024 + (size_t)stages * I8P_SUB * (I8P_A_BYTES + bn / 2 * I8P_BK) + sizeof(Int8SplitBarriers); }

template <typename OutT, int S>
__global__ void __cluster_dims__(2 * S, 1, 1) __launch_bounds__(I8P_THREADS, 1)
    int8_split_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Int8SplitParams pp) {
    extern __shared__ uint8_t i8s_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8s_smem_raw) + 1023) & ~(uintptr_t)1023);
    const Int8Product& p = pp.p;
    uint8_t* a_stages = smem;
    const int stages = pp.stages, b_bytes = pp.bn / 2 * I8P_BK;
    uint8_t* b_stages = smem + stages * I8P_SUB * I8P_A_BYTES;
    Int8SplitBarriers* bars = reinterpret_cast<Int8SplitBarriers*>(b_stages + stages * I8P_SUB * b_bytes);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank(), half = rank & 1u, leader = rank & ~1u;
    const int q = (int)(rank >> 1);  // which part of k
    const int tile = blockIdx.x / (2 * S), tn = tile / pp.tiles_m, row0 = (tile - tn * pp.tiles_m) * pp.bn;
    const int toks = min(pp.bn, p.rows - row0), cols = tile_columns(toks);
    const int nkb = (p.k + I8P_BK - 1) / I8P_BK, kb0 = nkb * q / S, kbs = nkb * (q + 1) / S - kb0;
    const int nst = (kbs + I8P_SUB - 1) / I8P_SUB;
    const auto pieces = [&](int st) { return min(I8P_SUB, kbs - st * I8P_SUB); };
    const uint32_t piece_bytes = 2u * (I8P_A_BYTES + (uint32_t)b_bytes);

    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        mbar_init(&bars->done, 1);
        mbar_init_fence();
    }
    if (warp == 2) tmem_alloc_pair(&bars->tmem_base, I8S_TOKENS);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);

    bool ok = true;
    if (warp == 0) {
        // ---------------- TMA ----------------
        const uint32_t full0 = map_to_rank(&bars->full[0], leader);
        const int row = tn * 2 * I8P_ROWS + (int)half * I8P_ROWS, token = row0 + (int)half * (cols / 2);
        const int early = min(stages, nst);  // the weights are no launch's work
        if (elect_one()) {
            for (int i = 0; i < early; ++i) {
                if (half == 0) mbar_arrive_expect_tx(&bars->full[i], pieces(i) * piece_bytes);
                for (int j = 0; j < pieces(i); ++j)
                    tma_load_2d_pair(a_stages + (size_t)(i * I8P_SUB + j) * I8P_A_BYTES, &tmap_w, (kb0 + i * I8P_SUB + j) * I8P_BK, row, full0 + 8u * i);
            }
        }
        __syncwarp();
        grid_dependency_wait();
        grid_launch_dependents();
        int s = 0, g = 0;
        uint32_t ph = 1;
        for (; g < nst; ++g) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars->empty[s], ph));
            if (!ok) {
                if (lane == 0) record_failure(p.status, STATUS_WAIT_EMPTY_TIMEOUT, g);
                break;
            }
            if (elect_one()) {
                if (g >= early && half == 0) mbar_arrive_expect_tx(&bars->full[s], pieces(g) * piece_bytes);
                for (int j = 0; j < pieces(g); ++j) {
                    const int at = s * I8P_SUB + j, k = (kb0 + g * I8P_SUB + j) * I8P_BK;
                    if (g >= early) tma_load_2d_pair(a_stages + (size_t)at * I8P_A_BYTES, &tmap_w, k, row, full0 + 8u * s);
                    tma_load_2d_pair(b_stages + (size_t)at * b_bytes, &tmap_x, k, token, full0 + 8u * s);
                }
            }
            __syncwarp();
            if (++s == stages) {
                s = 0;
                ph ^= 1u;
            }
        }
        if (!ok && half == 0) {  // the last copies are counted on the leader's barriers
            for (int i = 0; i < min(g, stages); ++i) {
                if (s == 0) { s = stages - 1; ph ^= 1u; } else --s;
                if (!mbar_wait_bounded(&bars->full[s], ph ^ 1u)) {
                    if (lane == 0) record_failure(p.status, STATUS_WAIT_DRAIN_TIMEOUT, i);
                    break;
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA ----------------
        if (half == 0) {
            const uint64_t da0 = make_smem_desc_sw128(smem_u32(a_stages)), db0 = make_smem_desc_sw128(smem_u32(b_stages));
            const uint32_t idesc = make_idesc_i8(2 * I8P_ROWS, cols);
            const unsigned short both = (unsigned short)(3u << leader);
            int s = 0;
            uint32_t ph = 0;
            for (int g = 0; g < nst; ++g) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars->full[s], ph));
                if (!ok) {
                    if (lane == 0) record_failure(p.status, STATUS_WAIT_FULL_TIMEOUT, g);
                    break;
                }
                tc_fence_after();
                const uint64_t da = da0 + (uint64_t)(s * I8P_SUB * (I8P_A_BYTES >> 4)), db = db0 + (uint64_t)(s * I8P_SUB * (b_bytes >> 4));
                if (elect_one()) {
                    for (int j = 0; j < pieces(g); ++j) {
                        const uint64_t dja = da + (uint64_t)(j * (I8P_A_BYTES >> 4)), djb = db + (uint64_t)(j * (b_bytes >> 4));
#pragma unroll
                        for (int k = 0; k < I8P_BK / 32; ++k) tc_mma_i8_pair(tmem_base, dja + 2 * k, djb + 2 * k, idesc, (g > 0 || j > 0 || k > 0) ? 1u : 0u);
                    }
                    tc_commit_pair_to(&bars->empty[s], both);
                    if (g == nst - 1) tc_commit_pair_to(&bars->done, both);
                }
                __syncwarp();
                if (++s == stages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
    } else if (warp >= 4) {
        grid_dependency_wait();
        if (!mbar_wait_bounded(&bars->done, 0)) {
            record_failure(p.status, STATUS_WAIT_MMA_TIMEOUT, 0);
            ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
    }
    __syncwarp();
    cluster_sync();  // every pair's products are done: the stages are free to take sums

    // 32 tokens at a time: those of chunk i are finished by pair i % S; the others send theirs to the CTA there with the same rows
    const int quarter = warp & 3, turn = (warp - 4) >> 2, chunks = cols / 32;
    const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const int slots = (chunks + S - 1) / S;  // chunks of a pair
    int* sums = reinterpret_cast<int*>(smem);  // [S - 1 senders][slots][32 tokens][128 rows]
    if (warp >= 4 && ok) {
        for (int c = turn; c < chunks; c += I8P_EPILOGUE / 4) {
            const int owner = c % S;
            if (owner == q) continue;
            uint32_t acc[32];
            tmem_ld_32x32(taddr + 32 * c, acc);
            const int sender = q < owner ? q : q - 1;
            const uint32_t dst = map_to_rank(sums + (sender * slots + c / S) * I8S_CHUNK + quarter * 32 + lane, 2 * owner + half);
#pragma unroll
            for (int j = 0; j < 32; ++j)
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst + 4u * I8P_ROWS * j), "r"(acc[j]) : "memory");
        }
    }
    __syncwarp();
    cluster_sync();
    if (warp >= 4 && ok) {
        const int n = tn * 2 * I8P_ROWS + (int)half * I8P_ROWS + quarter * 32 + lane;
        const float ws = n < p.n ? p.ws[n] : 0.0f;
        for (int c = q + S * turn; c < chunks; c += S * (I8P_EPILOGUE / 4)) {
            const int tok = 32 * c;
            const float xs = tok + lane < toks ? p.xs[row0 + tok + lane] : 0.0f;
            uint32_t acc[32];
            tmem_ld_32x32(taddr + tok, acc);
#pragma unroll
            for (int i = 0; i < S - 1; ++i) {
                const int* part = sums + (i * slots + c / S) * I8S_CHUNK + quarter * 32 + lane;
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[j] += (uint32_t)part[j * I8P_ROWS];
            }
            OutT* dst = static_cast<OutT*>(p.y) + (long long)(row0 + tok) * p.ldy + n;
            const int here = n < p.n ? toks - tok : 0;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                const float v = (float)(int)acc[j] * __shfl_sync(0xffffffffu, xs, j) * ws;
                if (j < here) *dst = from_float<OutT>(v);
                dst += p.ldy;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 2) tmem_dealloc_pair(tmem_base, I8S_TOKENS);
}

// How many clusters of the kernel the device holds at once; asked once per device, by whichever threads call first.
template <auto kernel> static int clusters_at_once(int ctas, size_t smem) {
    static std::atomic<int> known[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    int n = known[dev].load();
    if (n == 0) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)ctas, 1, 1);
        cfg.blockDim = dim3(I8P_THREADS, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)ctas;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            n = 0;
        }
        n = n > 0 ? n : -1;
        known[dev].store(n);
    }
    return n > 0 ? n : 0;
}

template <typename OutT, int S> static int split_t(const Int8Product& p, int bn, cudaStream_t s, bool dependent) {
    Int8SplitParams pp{};
    pp.p = p;
    pp.bn = bn;
    pp.tiles_m = (p.rows + bn - 1) / bn;
    const int tiles = (p.n + 2 * I8P_ROWS - 1) / (2 * I8P_ROWS) * pp.tiles_m;
    constexpr auto kernel = int8_split_kernel<OutT, S>;
    cudaError_t e = allow_full_smem<kernel>();
    if (e != cudaSuccess) return set_error((int)e, cudaGetErrorString(e));
    if (tiles > clusters_at_once<kernel>(2 * S, (size_t)runtime_info().smem_optin - 1024)) return B200Q_ERR_UNSUPPORTED;
    pp.stages = I8P_MAX_STAGES;
    while (i8s_smem(pp.stages, bn) > (size_t)runtime_info().smem_optin - 1024) --pp.stages;
    CUtensorMap map_w, map_x;
    if (!int8_pair_maps(p, bn, &map_w, &map_x)) return set_error(B200Q_ERR_INVALID, "no tensor map for these rows");
    e = launch_kernel(kernel, dim3((unsigned)tiles * 2 * S, 1, 1), I8P_THREADS, i8s_smem(pp.stages, bn), s, dependent, map_w, map_x, pp);
    return e == cudaSuccess ? B200Q_OK : set_error((int)e, cudaGetErrorString(e));
}
template <typename OutT> static int split_out(const Int8Product& p, cudaStream_t s, bool dependent) {
    const int tiles_n = (p.n + 2 * I8P_ROWS - 1) / (2 * I8P_ROWS), pairs = runtime_info().sm_count / 2;
    const int tiles_m = (p.rows + I8S_TOKENS - 1) / I8S_TOKENS, bn = ((p.rows + tiles_m - 1) / tiles_m + 31) & ~31;
    const int nkb = (p.k + I8P_BK - 1) / I8P_BK;
    if (nkb < I8S_LEAST || 2LL * tiles_n * tiles_m > pairs) return B200Q_ERR_UNSUPPORTED;
    if (4 * tiles_n * tiles_m <= pairs) {
        const int rc = split_t<OutT, 4>(p, bn, s, dependent);
        if (rc != B200Q_ERR_UNSUPPORTED) return rc;
    }
    return split_t<OutT, 2>(p, bn, s, dependent);
}
int int8_product_split(int elem, const Int8Product& p, cudaStream_t s, bool dependent) {
    if (p.experts > 1 || p.offsets != nullptr || p.act != INT8_ACT_NONE) return B200Q_ERR_UNSUPPORTED;
    if (elem == ELEM_F32) return split_out<float>(p, s, dependent);
    if (elem == ELEM_F16) return split_out<__half>(p, s, dependent);
    return split_out<__nv_bfloat16>(p, s, dependent);
}

}  // namespace b200q
