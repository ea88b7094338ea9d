// Products of int8 rows on warp-level integer MMAs, for few tokens: what they cost is reading the weights, once, from HBM straight into MMA
// fragments. One to eight warps of a CTA share a tile of 16 or 32 weight rows and 8 or 16 tokens, each a part of k, and add up through
// shared memory; the sums are integers, so their order changes nothing.
//
// A lane loads 16 neighbouring bytes of a row: of the four words two make its part of one 32-k MMA and two that of the next. That takes
// the k of a 64-byte piece in another order than they lie, the same one for weights and tokens, which a sum does not mind.
//
// The CTAs are persistent and a warp's loads run one batch of pieces ahead of its products, across the border from one tile to the next:
// 64 KB on their way per SM all the time. (CTAs of one tile each, without that: 14336 x 4096 by one token 24.9 us against 13.4, 4096 x
// 28672 24.1 against 20.3 of which HBM needs 18.)
#include "int8.cuh"

namespace b200q {

constexpr int I8R_WARPS = 8;
constexpr int I8R_STEP = 64;  // k of one piece
constexpr int I8R_PER_SM = 2; // CTAs on an SM

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

// A lane's words of U pieces of 16 R weight rows and 8 NT tokens. Pieces from `steps` on, and lanes beyond the row's end, count as zeros.
template <int R, int NT, int U, int WK> struct RowPieces {
    uint4 a[U][2 * R], b[U][NT];
    __device__ __forceinline__ void load_weights(const int8_t* const (&w)[2 * R], int step, int kp, int t) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k0 = (step + u * WK) * I8R_STEP;
#pragma unroll
            for (int i = 0; i < 2 * R; ++i) a[u][i] = k0 + 16 * t < kp ? ldg_stream(w[i] + k0) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    __device__ __forceinline__ void load_tokens(const int8_t* const (&x)[NT], int step, int kp, int t) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k0 = (step + u * WK) * I8R_STEP;
#pragma unroll
            for (int j = 0; j < NT; ++j) b[u][j] = k0 + 16 * t < kp ? *reinterpret_cast<const uint4*>(x[j] + k0) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    __device__ __forceinline__ void multiply(int (&acc)[R][NT][4]) const {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    mma_s8(acc[i][j], a[u][2 * i].x, a[u][2 * i + 1].x, a[u][2 * i].y, a[u][2 * i + 1].y, b[u][j].x, b[u][j].y);
                    mma_s8(acc[i][j], a[u][2 * i].z, a[u][2 * i + 1].z, a[u][2 * i].w, a[u][2 * i + 1].w, b[u][j].z, b[u][j].w);
                }
    }
};

template <typename OutT, int R, int NT, int U, int WK>
__global__ void __launch_bounds__(32 * I8R_WARPS, I8R_PER_SM) int8_rows_kernel(const Int8Product p) {
    constexpr int ROWS = 16 * R, TOKENS = 8 * NT, PITCH = ROWS + 4, GROUPS = I8R_WARPS / WK;
    __shared__ int sums[I8R_WARPS][TOKENS][PITCH];
    extern __shared__ int lists[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = warp / WK, wk = warp % WK;
    const int kp = (p.k + 15) & ~15, steps = (kp + I8R_STEP - 1) / I8R_STEP, batches = (steps + U * WK - 1) / (U * WK);
    Int8TileList list{};
    list.build<32 * I8R_WARPS>(p, TOKENS, (p.n + ROWS - 1) / ROWS, lists);
    Int8TileList ahead = list;

    // Loads run a batch ahead of the products, and on into the next tile.
    RowPieces<R, NT, U, WK> now, next;
    const int8_t *w[2 * R], *x[NT];
    const int first_tile = blockIdx.x + gridDim.x * group, tile_step = gridDim.x * GROUPS;
    int ahead_tile = first_tile, ahead_batch = 0;
    const auto aim = [&] {
        const Int8Tile at = ahead.find(ahead_tile, lane);
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) w[i] = p.wq + ((long long)at.e * p.n + min(at.tn * ROWS + 8 * i + g, p.n - 1)) * p.ldw + 16 * t;
#pragma unroll
        for (int j = 0; j < NT; ++j) x[j] = p.xq + (long long)(at.row0 + min(8 * j + g, at.toks - 1)) * p.ldx + 16 * t;
    };
    const auto advance = [&] {
        if (++ahead_batch < batches) return;
        ahead_batch = 0;
        ahead_tile += tile_step;
        if (ahead_tile < list.ntiles) aim();
    };
    const auto fill = [&](RowPieces<R, NT, U, WK>& pieces) {
        if (ahead_tile >= list.ntiles) return;
        pieces.load_weights(w, ahead_batch * U * WK + wk, kp, t);
        pieces.load_tokens(x, ahead_batch * U * WK + wk, kp, t);
        advance();
    };
    if (ahead_tile < list.ntiles) {
        aim();
        now.load_weights(w, wk, kp, t);  // the weights are no launch's work: on their way before the rows are there
    }
    grid_dependency_wait();
    grid_launch_dependents();
    if (ahead_tile < list.ntiles) {
        now.load_tokens(x, wk, kp, t);
        advance();
    }
    bool flip = false;
    for (int tile = first_tile; tile < list.ntiles; tile += tile_step) {
        int acc[R][NT][4] = {};
        for (int b = 0; b < batches; ++b) {
            if (!flip) {
                fill(next);
                now.multiply(acc);
            } else {
                fill(now);
                next.multiply(acc);
            }
            flip = !flip;
        }
        const Int8Tile at = list.find(tile, lane);
        const int row0 = at.tn * ROWS;
        const float* ws = p.ws + (long long)at.e * p.n + row0;
        const float* xs = p.xs + at.row0;
        OutT* y = static_cast<OutT*>(p.y) + (long long)at.row0 * p.ldy;
        const auto put = [&](int tok, int r, int sum) {  // row r of the tile
            if (row0 + r < p.n) y[tok * p.ldy + row0 + r] = from_float<OutT>((float)sum * xs[tok] * ws[r]);
        };
        const auto put_gated = [&](int tok, int r, int gate, int up) {  // r: the gate's row, up is 8 rows on
            const int col = row0 / 2 + (r >> 4) * 8 + (r & 7);
            if (col < p.n_out) y[tok * p.ldy + col] = from_float<OutT>(int8_activate((float)gate * xs[tok] * ws[r], p.act) * ((float)up * xs[tok] * ws[r + 8]));
        };
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) sums[warp][8 * j + 2 * t + (c & 1)][16 * i + g + 8 * (c >> 1)] = acc[i][j][c];
        named_bar_sync(1 + group, 32 * WK);
        const auto total = [&](int tok, int r) {
            int sum = 0;
#pragma unroll
            for (int v = 0; v < WK; ++v) sum += sums[group * WK + v][tok][r];
            return sum;
        };
        const int member = wk * 32 + lane;
        if (p.act == INT8_ACT_NONE) {
            for (int i = member; i < at.toks * ROWS; i += 32 * WK) put(i / ROWS, i % ROWS, total(i / ROWS, i % ROWS));
        } else {
            for (int i = member; i < at.toks * ROWS / 2; i += 32 * WK) {
                const int c = i % (ROWS / 2), tok = i / (ROWS / 2), r = (c & ~7) * 2 + (c & 7);
                put_gated(tok, r, total(tok, r), total(tok, r + 8));
            }
        }
        named_bar_sync(1 + group, 32 * WK);
    }
}

template <typename OutT, int R, int NT, int U, int WK> static cudaError_t rows_launch(const Int8Product& p, cudaStream_t s, bool dependent) {
    // at most one group of tokens more per expert than the rows fill
    const long long tiles = (long long)((p.n + 16 * R - 1) / (16 * R)) * ((p.rows + 8 * NT - 1) / (8 * NT) + p.experts - 1), fit = (long long)I8R_PER_SM * runtime_info().sm_count;
    return launch_kernel(int8_rows_kernel<OutT, R, NT, U, WK>, dim3((unsigned)(tiles < fit ? tiles : fit), 1, 1), 32 * I8R_WARPS, int8_list_bytes(p.experts), s, dependent, p);
}
// Which form of the kernel takes a product; none where the tensor-core kernels (int8_pair.cu, int8_split.cu) are the faster ones. What
// decides is how the tiles of 16 rows fill the places that the SMs have for CTAs (two each, 296 on 148), and how many tokens meet each
// weight: a tile more than the places are, and some SM has twice the work. us, quantizer included, bf16, weights out of HBM (tc: the
// tensor-core kernels):
//   up to 8 tokens   8 warps a tile while every tile has a place, then 4 (two tiles a CTA): of 14336 k 296 tiles 14.0 (4: 16.5), 304 18.0
//                    (16.8), 448 20.2 (19.5); of 4096 k 6.2 (6.9), 7.7 (7.1), 8.3 (8.1); of 1024 k 3.9 (3.9), 4.5 (3.9), 4.9 (4.3). 4 warps
//                    up to four tiles a place, then 2 warps and 32 rows: of 14336 k 1184 tiles 42.9 (2: 47.0), 1200 48.7 (47.3), 1792
//                    68.7 (64.5); of 4096 k 14.9 (17.0), 16.4 (17.1), 21.7 (21.1); of 1024 k 6.6 (6.5), 7.1 (6.7), 9.0 (7.9)
//                    experts: one token through 2 of 8 of 4096 x 14336, 4 warps for the 512 tiles of down 68.9 (8: 72.7); 16 tokens through
//                    8 of 128 of 2048 x 768 67.8 with 2 (4 warps 78.2, tc 73.5). Experts with five to eight tokens, of which some have
//                    more: 4 warps up to six tiles a place, then tc (20 tokens through 1 of 4 of 1024 x 2400, 1200 tiles, 17.2 and 19.2; 10
//                    through 2 of 4 of 4096 x 3500, 1752 tiles, 41 and 61, but 24 through 4 of 16 of 2048 x 800, 1600 tiles, 30.9 and 28.8;
//                    48 through 6 of 64 of 2048 x 1408, 11264 tiles, 98.5 and 97.8)
//   more, 16 at once a group is 16 tokens of a tile. Of long rows as many groups as places: 16 tokens of 14336 k 288 groups 15.6 (tc
//                    17.6), 320 23.9 (18.6); of 8192 k 11.1 (13.3), 15.8 (13.9). Of rows up to 6144 twice as many: of 6144 k 288 9.1 (11.7),
//                    320 12.7 (12.2), 513 14.2 (14.5), 640 18.1 (16.6); of 4096 k 513 10.7 (12.2), 640 13.4 (13.2)
//                    with more groups than places and more than 16 tokens, 32 rows a tile: 32 tokens of 4096 k 512 groups 8.6 (16 rows 9.7,
//                    tc 10.1), 640 13.2 (tc 10.7)
enum class RowsForm { none, few_tiles, some_tiles, many_tiles, tokens16, tokens32 };
static RowsForm rows_form(const Int8Product& p) {
    const int used = p.experts < p.rows ? p.experts : p.rows;  // experts with tokens, at most
    const int per = (p.rows + used - 1) / used;
    const long long tiles = (long long)((p.n + 15) / 16) * used;
    const long long places = (long long)I8R_PER_SM * runtime_info().sm_count;
    if (per <= 8 && tiles <= (p.experts > 1 && per > 4 ? 6 : 4) * places) return tiles <= places ? RowsForm::few_tiles : RowsForm::some_tiles;
    if (per <= (p.experts > 1 ? 4 : 8)) return RowsForm::many_tiles;
    const long long groups = (per + 15) / 16 * tiles;
    if (groups <= (p.k > 6144 ? places : 2 * places)) return groups <= places || per <= 16 ? RowsForm::tokens16 : RowsForm::tokens32;
    return RowsForm::none;
}
bool int8_rows_pays(const Int8Product& p) { return rows_form(p) != RowsForm::none; }

template <typename OutT> static cudaError_t rows_t(const Int8Product& p, cudaStream_t s, bool dependent) {
    switch (rows_form(p)) {
        case RowsForm::few_tiles: return rows_launch<OutT, 1, 1, 4, 8>(p, s, dependent);
        case RowsForm::some_tiles: return rows_launch<OutT, 1, 1, 4, 4>(p, s, dependent);
        case RowsForm::many_tiles: return rows_launch<OutT, 2, 1, 2, 2>(p, s, dependent);
        case RowsForm::tokens16: return rows_launch<OutT, 1, 2, 2, 8>(p, s, dependent);
        default: return rows_launch<OutT, 2, 2, 1, 8>(p, s, dependent);
    }
}

cudaError_t int8_product_rows(int elem, const Int8Product& p, cudaStream_t s, bool dependent) {
    if (elem == ELEM_F32) return rows_t<float>(p, s, dependent);
    if (elem == ELEM_F16) return rows_t<__half>(p, s, dependent);
    return rows_t<__nv_bfloat16>(p, s, dependent);
}

}  // namespace b200q
