// What the tensor-core kernels of int8 products share (int8_pair.cu: tile after tile; int8_split.cu: few tiles, k divided).
#pragma once
#include <cuda.h>

#include "int8.cuh"
#include "tcgen05.cuh"

namespace b200q {

constexpr int I8P_ROWS = 128;      // weight rows of one CTA = TMEM lanes
constexpr int I8P_TOKENS = 256;    // tokens of a tile at most = TMEM columns of one accumulator
constexpr int I8P_BK = 128;        // k per stage: one 128-byte swizzled row
constexpr int I8P_SUB = 2;         // such pieces per stage: the hand-over of a stage from TMA to tensor core and back takes as long as a
                                   // small tile's products of 128 k (16 tokens, 16384 k: 345 cycles per 128 k with one, 275 with two)
constexpr int I8P_MAX_STAGES = 6;
constexpr int I8P_A_BYTES = I8P_ROWS * I8P_BK;
constexpr int I8P_THREADS = 384;   // warp 0 TMA, warp 1 MMA, warp 2 TMEM, warps 4-11 epilogue
constexpr int I8P_EPILOGUE = 8;    // warps: two to a quarter of the TMEM lanes, taking its columns 32 at a time in turn


__device__ __forceinline__ int tile_columns(int toks) { return (toks + 31) & ~31; }  // N of the instruction

// Tensor maps of the weights, in boxes of 128 rows, and of the activations, in boxes of half a tile's tokens.
static bool int8_pair_maps(const Int8Product& p, int bn, CUtensorMap* w, CUtensorMap* x) {
    const cuuint64_t kp = (cuuint64_t)((p.k + 15) & ~15), wdims[2] = {kp, (cuuint64_t)p.experts * p.n}, xdims[2] = {kp, (cuuint64_t)p.rows};
    const cuuint32_t wbox[2] = {I8P_BK, I8P_ROWS}, xbox[2] = {I8P_BK, (cuuint32_t)(bn / 2)};
    return encode_tiled_2d_cached(w, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.wq, wdims, (cuuint64_t)p.ldw, wbox, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ==
               CUDA_SUCCESS &&
           encode_tiled_2d_cached(x, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.xq, xdims, (cuuint64_t)p.ldx, xbox, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ==
               CUDA_SUCCESS;
}

// int8_split.cu: B200Q_ERR_UNSUPPORTED where it is not the faster one
int int8_product_split(int elem, const Int8Product& p, cudaStream_t s, bool dependent);

}  // namespace b200q
