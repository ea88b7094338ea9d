// Products of int8 rows on the tensor cores: tcgen05.mma.cta_group::2, kind::i8. A pair of SMs owns a tile of 256 weight rows x up to 256
// tokens; each SM holds 128 of the weight rows and half of the tokens in shared memory, brought there by TMA in 128-byte pieces of k,
// and the sums stay in tensor memory as 32-bit integers until the epilogue scales them by token and channel.
//
// The weights sit on the M side of the instruction: its N side, the tokens, goes in steps of 32, so a ragged number of tokens wastes
// little. With several matrices (experts) the tiles of all of them form one list, and a tile holds rows of one expert; where an expert's
// rows begin and end is read on the device. A tile's boxes may reach into the next expert's rows: those columns are computed and not
// stored. Two accumulators: the epilogue of one tile runs beside the product of the next.
//
// Every wait is bounded; a wait that gives up records a code in the device status word, work is skipped, and the kernel still frees its
// TMEM columns before it returns.
#include "int8_pair.cuh"

namespace b200q {

constexpr int I8P_TMEM_COLS = 512;  // two accumulators

struct Int8PairParams {
    Int8Product p;
    int bn;       // tokens per tile at most: a multiple of 32
    int stages;
    int tiles_n;  // weight tiles of 256 rows, of one matrix
};
struct Int8PairBarriers {
    uint64_t full[I8P_MAX_STAGES], empty[I8P_MAX_STAGES];
    uint64_t tmem_full[2], tmem_empty[2];
    uint32_t tmem_base, unused[3];
    float xs[I8P_EPILOGUE][I8P_TOKENS / (I8P_EPILOGUE / 4)];  // an epilogue warp's token scales of its tile
};
static size_t i8p_smem(int stages, int bn, int experts) {
    return 1024 + (size_t)stages * I8P_SUB * (I8P_A_BYTES + bn / 2 * I8P_BK) + sizeof(Int8PairBarriers) + int8_list_bytes(experts);
}

// The first `count` of N values, to consecutive rows. (By whole warps.)
template <int N, typename OutT> __device__ __forceinline__ void store_column(OutT* dst, long long ld, const float* v, int count) {
    if (__all_sync(0xffffffffu, count >= N)) {
#pragma unroll
        for (int j = 0; j < N; ++j) dst[j * ld] = from_float<OutT>(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < count) dst[j * ld] = from_float<OutT>(v[j]);
    }
}

template <typename OutT, int ACT>  // ACT: INT8_ACT_NONE, or the activation of a gated product
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8P_THREADS, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const Int8PairParams pp) {
    extern __shared__ uint8_t i8p_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(i8p_smem_raw) + 1023) & ~(uintptr_t)1023);
    const Int8Product& p = pp.p;
    uint8_t* a_stages = smem;
    const int stages = pp.stages, half = pp.bn / 2, b_bytes = half * I8P_BK;  // bytes: a multiple of 1024
    uint8_t* b_stages = smem + stages * I8P_SUB * I8P_A_BYTES;
    Int8PairBarriers* bars = reinterpret_cast<Int8PairBarriers*>(b_stages + stages * I8P_SUB * b_bytes);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const int nkb = (p.k + I8P_BK - 1) / I8P_BK;
    const uint32_t piece_bytes = 2u * (I8P_A_BYTES + (uint32_t)b_bytes);  // both CTAs' operands of a piece
    const int nst = (nkb + I8P_SUB - 1) / I8P_SUB;
    const auto pieces = [&](int st) { return min(I8P_SUB, nkb - st * I8P_SUB); };

    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&bars->full[s], 1);
            mbar_init(&bars->empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bars->tmem_full[s], 1);
            mbar_init(&bars->tmem_empty[s], 2 * I8P_EPILOGUE);
        }
        mbar_init_fence();
    }
    if (warp == 2) tmem_alloc_pair(&bars->tmem_base, I8P_TMEM_COLS);
    Int8TileList list{};
    list.build<I8P_THREADS>(p, pp.bn, pp.tiles_n, reinterpret_cast<int*>(bars + 1));
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the other CTA's barriers exist before anything arrives at them
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
    const int ntiles = list.ntiles;
    if (warp == 0) {
        // ---------------- TMA: this CTA's 128 weight rows and half of the tokens; the leader's barrier counts both CTAs' bytes ----
        int s = 0, g = 0;
        uint32_t ph = 1;
        bool ok = true;
        const uint32_t full0 = map_to_rank(&bars->full[0], 0);
        // The weights are no launch's work: the first stages' are on their way before the rows are there.
        int early = 0;
        if ((p.offsets == nullptr || p.offsets_known) && pair < ntiles) {
            const Int8Tile t = list.find(pair, lane);
            const int row = t.e * p.n + t.tn * 2 * I8P_ROWS + (int)rank * I8P_ROWS;
            early = min(stages, nst);
            if (elect_one()) {
                for (int i = 0; i < early; ++i) {
                    if (rank == 0) mbar_arrive_expect_tx(&bars->full[i], pieces(i) * piece_bytes);
                    for (int j = 0; j < pieces(i); ++j)
                        tma_load_2d_pair(a_stages + (size_t)(i * I8P_SUB + j) * I8P_A_BYTES, &tmap_w, (i * I8P_SUB + j) * I8P_BK, row, full0 + 8u * i);
                }
            }
            __syncwarp();
        }
        grid_dependency_wait();
        grid_launch_dependents();
        for (int tile = pair; tile < ntiles && ok; tile += npairs) {
            const Int8Tile t = list.find(tile, lane);
            const int row = t.e * p.n + t.tn * 2 * I8P_ROWS + (int)rank * I8P_ROWS, token = t.row0 + (int)rank * (tile_columns(t.toks) / 2);
            for (int kb = 0; kb < nst; ++kb, ++g) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars->empty[s], ph));
                if (!ok) {
                    if (lane == 0) record_failure(p.status, STATUS_WAIT_EMPTY_TIMEOUT, g);
                    break;
                }
                if (elect_one()) {
                    if (g >= early && rank == 0) mbar_arrive_expect_tx(&bars->full[s], pieces(kb) * piece_bytes);
                    for (int j = 0; j < pieces(kb); ++j) {
                        const int at = s * I8P_SUB + j, k = (kb * I8P_SUB + j) * I8P_BK;
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
        }
        // the leader waits for its last copies before the CTAs may exit (they are counted on its barriers; the MMAs have
        // consumed them unless something gave up)
        if (!ok && rank == 0) {
            for (int q = 0; q < min(g, stages); ++q) {
                if (s == 0) { s = stages - 1; ph ^= 1u; } else --s;
                if (!mbar_wait_bounded(&bars->full[s], ph ^ 1u)) {
                    if (lane == 0) record_failure(p.status, STATUS_WAIT_DRAIN_TIMEOUT, q);
                    break;
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer: an elected lane of the leader, for both SMs ----------------
        if (rank == 0) {
            const uint64_t da0 = make_smem_desc_sw128(smem_u32(a_stages)), db0 = make_smem_desc_sw128(smem_u32(b_stages));
            int s = 0, ti = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int tile = pair; tile < ntiles && ok; tile += npairs, ++ti) {
                const int buf = ti & 1;
                const uint32_t idesc = make_idesc_i8(2 * I8P_ROWS, tile_columns(list.find(tile, lane).toks));
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars->tmem_empty[buf], ((ti >> 1) & 1) ^ 1));
                if (!ok) {
                    if (lane == 0) record_failure(p.status, STATUS_WAIT_MMA_TIMEOUT, 2000 + ti);
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem_base + buf * I8P_TOKENS;
                for (int kb = 0; kb < nst; ++kb) {
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars->full[s], ph));
                    if (!ok) {
                        if (lane == 0) record_failure(p.status, STATUS_WAIT_FULL_TIMEOUT, kb);
                        break;
                    }
                    tc_fence_after();
                    const uint64_t da = da0 + (uint64_t)(s * I8P_SUB * (I8P_A_BYTES >> 4)), db = db0 + (uint64_t)(s * I8P_SUB * (b_bytes >> 4));
                    if (elect_one()) {
                        for (int j = 0; j < pieces(kb); ++j) {
                            const uint64_t dja = da + (uint64_t)(j * (I8P_A_BYTES >> 4)), djb = db + (uint64_t)(j * (b_bytes >> 4));
#pragma unroll
                            for (int k = 0; k < I8P_BK / 32; ++k) tc_mma_i8_pair(d, dja + 2 * k, djb + 2 * k, idesc, (kb > 0 || j > 0 || k > 0) ? 1u : 0u);
                        }
                        tc_commit_pair(&bars->empty[s]);  // frees the stage in both CTAs when these MMAs have read it
                        if (kb == nst - 1) tc_commit_pair(&bars->tmem_full[buf]);
                    }
                    __syncwarp();
                    if (++s == stages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
        }
    } else if (warp >= 4) {
        // ---------------- epilogue: thread = weight row, 32 tokens at a time; a warp's store is 32 neighbouring outputs ----------------
        // A tile's scales are asked for when the one before is done, ahead of the wait for the product; those of the tokens go through
        // shared memory, four to a load, where a shuffle brought one. us, 8192 x 8192 bf16 outputs of 128 k / 2048 k: scales by shuffles and
        // after the wait 48.0 / 88.5, so 41.8 / 88.9; asked for while the tile before is at work 37.5 / 90.4, with 16 epilogue warps
        // 38.6 / 90.6, with the accumulator's next columns on their way as well 43.3 / 90.1, bf16 outputs gathered to 16 bytes in shared
        // memory 51.4 / 90.9.
        constexpr int STEP = 8 * I8P_EPILOGUE, CHUNKS = I8P_TOKENS / STEP;  // of a warp's 32 tokens, in a tile
        const int quarter = warp & 3, turn = (warp - 4) >> 2;
        grid_dependency_wait();
        float* scales = bars->xs[warp - 4];
        Int8Tile t{};
        float ws = 0.0f, xs[CHUNKS];
        const auto ask = [&](int tile) {
            if (tile >= ntiles) return;
            t = list.find(tile, lane);
            const int n = t.tn * 2 * I8P_ROWS + (int)rank * I8P_ROWS + quarter * 32 + lane;
            ws = n < p.n ? p.ws[(long long)t.e * p.n + n] : 0.0f;
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) {
                const int c = 32 * turn + i * STEP + lane;
                xs[i] = c < t.toks ? p.xs[t.row0 + c] : 0.0f;
            }
        };
        ask(pair);
        int ti = 0;
        for (int tile = pair; tile < ntiles; tile += npairs, ++ti) {
            const int buf = ti & 1, toks = t.toks, n = t.tn * 2 * I8P_ROWS + (int)rank * I8P_ROWS + quarter * 32 + lane;
            const float w = ws;
            OutT* y = static_cast<OutT*>(p.y) + (long long)t.row0 * p.ldy;
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) scales[32 * i + lane] = xs[i];
            bool ok = mbar_wait_bounded(&bars->tmem_full[buf], (ti >> 1) & 1);
            if (!ok) record_failure(p.status, STATUS_WAIT_MMA_TIMEOUT, ti);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * I8P_TOKENS;
            const auto finish = [&](const uint32_t (&acc)[32], int c) {
                float v[32];
                const float* sc = scales + c / STEP * 32;
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 x = *reinterpret_cast<const float4*>(sc + j);
                    v[j] = (float)(int)acc[j] * x.x * w;
                    v[j + 1] = (float)(int)acc[j + 1] * x.y * w;
                    v[j + 2] = (float)(int)acc[j + 2] * x.z * w;
                    v[j + 3] = (float)(int)acc[j + 3] * x.w * w;
                }
                OutT* dst = y + c * p.ldy;
                if constexpr (ACT == INT8_ACT_NONE) {
                    store_column<32>(dst + n, p.ldy, v, n < p.n ? toks - c : 0);
                } else {
                    // rows 8.. of 16 hold up, the others gate: the lane of a gate row takes tokens 0..15, that of its up row 16..31
                    const bool is_up = (lane & 8) != 0;
                    const int col = (n >> 4) * 8 + (n & 7), from = is_up ? 16 : 0;
                    // All sixteen before the first store: under a store's condition the compiler put each value's arithmetic in a branch
                    // of its own, one after the other (7696 rows of 60 experts, 256 -> 2 x 512 -> 256: 54.3 us the layer, now 44.1).
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float other = __shfl_xor_sync(0xffffffffu, is_up ? v[j] : v[16 + j], 8);
                        const float gate = is_up ? other : v[j], up = is_up ? v[16 + j] : other;
                        v[j] = int8_activate(gate, ACT) * up;
                        asm volatile("" : "+f"(v[j]));
                    }
                    store_column<16>(dst + from * p.ldy + col, p.ldy, v, col < p.n_out ? toks - c - from : 0);
                }
            };
            __syncwarp();  // the scales are there
            for (int c = 32 * turn; c < toks; c += STEP) {
                uint32_t acc[32];
                tmem_ld_32x32(taddr + c, acc);
                finish(acc, c);
            }
            ask(tile + npairs);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_rank(&bars->tmem_empty[buf], 0));  // the accumulator may be reused
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // neither CTA leaves while the other may still read its operands or arrive at its barriers
    if (warp == 2) tmem_dealloc_pair(tmem_base, I8P_TMEM_COLS);
}

// ---- host side -------------------------------------------------------------------------------------------------------------------
// Tokens per tile. One matrix: the height with the least waves x height, as tiles go out in waves of one per CTA pair; a wave takes as
// long as its tile is high, but no less than a tile of about 148 tokens, and some 24 tokens' worth to fill and drain. Several: a bit
// more than an expert has on average.
static int int8_token_tile(const Int8Product& p, int tiles_n) {
    if (p.experts > 1) {
        const int per = p.rows / p.experts, bn = (per + per / 4 + 16 + 31) & ~31;
        return bn < I8P_TOKENS ? bn : I8P_TOKENS;
    }
    const int pairs = runtime_info().sm_count / 2;
    long long best = 0;
    int best_bn = 0;
    for (int tm = (p.rows + I8P_TOKENS - 1) / I8P_TOKENS, last = 0;; ++tm) {
        const int bn = (((p.rows + tm - 1) / tm) + 31) & ~31;
        if (best_bn != 0 && bn < 128) break;
        if (bn == last) continue;
        last = bn;
        const long long waves = ((long long)((p.rows + bn - 1) / bn) * tiles_n + pairs - 1) / pairs;
        const long long cost = waves * ((bn > 148 ? bn : 148) + 24);
        if (best_bn == 0 || cost * 100 < best * 95) {
            best = cost;
            best_bn = bn;
        }
    }
    return best_bn;
}

template <typename OutT, int ACT> static int pair_t(const Int8Product& p, cudaStream_t s, bool dependent) {
    Int8PairParams pp{};
    pp.p = p;
    pp.tiles_n = (p.n + 2 * I8P_ROWS - 1) / (2 * I8P_ROWS);
    pp.bn = int8_token_tile(p, pp.tiles_n);
    pp.stages = I8P_MAX_STAGES;
    while (i8p_smem(pp.stages, pp.bn, p.experts) > (size_t)runtime_info().smem_optin - 1024) --pp.stages;
    CUtensorMap map_w, map_x;
    if (!int8_pair_maps(p, pp.bn, &map_w, &map_x)) return set_error(B200Q_ERR_INVALID, "no tensor map for these rows");
    constexpr auto kernel = int8_pair_kernel<OutT, ACT>;
    cudaError_t e = allow_full_smem<kernel>();
    if (e == cudaSuccess) {
        const int pairs = runtime_info().sm_count / 2;
        // at most one tile more per expert than the rows fill
        const long long tiles = ((long long)p.rows / pp.bn + p.experts) * pp.tiles_n;
        const unsigned grid = 2u * (unsigned)(tiles < pairs ? tiles : pairs);
        e = launch_kernel(kernel, dim3(grid, 1, 1), I8P_THREADS, i8p_smem(pp.stages, pp.bn, p.experts), s, dependent, map_w, map_x, pp);
    }
    return e == cudaSuccess ? B200Q_OK : set_error((int)e, cudaGetErrorString(e));
}
template <typename OutT> static int pair_out(const Int8Product& p, cudaStream_t s, bool dependent) {
    switch (p.act) {
        case INT8_ACT_NONE: return pair_t<OutT, INT8_ACT_NONE>(p, s, dependent);
        case INT8_ACT_GELU: return pair_t<OutT, INT8_ACT_GELU>(p, s, dependent);
        case INT8_ACT_RELU: return pair_t<OutT, INT8_ACT_RELU>(p, s, dependent);
        case INT8_ACT_GELU_ERF: return pair_t<OutT, INT8_ACT_GELU_ERF>(p, s, dependent);
        case INT8_ACT_SIGMOID: return pair_t<OutT, INT8_ACT_SIGMOID>(p, s, dependent);
        default: return pair_t<OutT, INT8_ACT_SILU>(p, s, dependent);
    }
}

bool int8_pair_ready() { return encode_tiled_fn() != nullptr; }

int int8_product_pair(int elem, const Int8Product& p, cudaStream_t s, bool dependent) {
    const int rc = int8_product_split(elem, p, s, dependent);
    if (rc != B200Q_ERR_UNSUPPORTED) return rc;
    if (elem == ELEM_F32) return pair_out<float>(p, s, dependent);
    if (elem == ELEM_F16) return pair_out<__half>(p, s, dependent);
    return pair_out<__nv_bfloat16>(p, s, dependent);
}

}  // namespace b200q
