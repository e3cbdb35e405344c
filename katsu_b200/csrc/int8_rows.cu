// The 8-bit product for a few tokens (m <= 8): the weights are read once, 16 bytes a lane, and multiplied on the CUDA cores
// four values an instruction (dp4a).
//
// A block holds the tokens' rows in shared memory, in 8 bits, and quantises them itself where x comes in f32, so that one
// token's product is one launch.  A warp takes two rows of the weights; where there are fewer pairs of rows than warps on
// the GPU, up to eight warps of a block share a pair and cut k among them.  Bound: the weights' bytes at HBM (or L2) rate.
#include "int8.cuh"

namespace {

constexpr int kWarps = 8, kRows = 2, kUnroll = 4;
constexpr size_t kMostShared = size_t(200) * 1024;  // a block's tokens

template <int M>
__global__ void __launch_bounds__(kWarps * 32) int8_rows_kernel(const float *__restrict__ x, const int8_t *__restrict__ xq,
                                                                const float *__restrict__ xs, const int8_t *__restrict__ wq,
                                                                const float *__restrict__ ws, const float *bias, float *y,
                                                                int m, int k, int n, int pitch, int share) {
    extern __shared__ __align__(16) unsigned char tokens[];  // [M][pitch]
    __shared__ float largest[M][kWarps];
    __shared__ float scales[M];
    __shared__ int sums[kWarps][kRows * M];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    launch_next();
    launch_wait();
    const int pairs = (n + kRows - 1) / kRows, per_block = kWarps / share, part = warp % share;
    const int units = pitch / 16, begin = int((long long)units * part / share), end = int((long long)units * (part + 1) / share);
    // 16 bytes a lane of the pair's rows, kUnroll times: all on their way before the first is used
    int4 v[kUnroll][kRows];
    auto fetch = [&](int pair, int u0) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int4 *w = reinterpret_cast<const int4 *>(wq + size_t(min(pair * kRows + r, n - 1)) * pitch);
#pragma unroll
            for (int q = 0; q < kUnroll; ++q)
                v[q][r] = pair < pairs && u0 + 32 * q < end ? __ldg(w + u0 + 32 * q) : make_int4(0, 0, 0, 0);
        }
    };
    fetch(blockIdx.x * per_block + warp / share, begin + lane);  // the first ones while the tokens are quantised
    // ---- the tokens ----
    if (x != nullptr) {
        const bool vec = (k & 3) == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
        auto load4 = [&](int i, int j, float (&v)[4]) {
            const float *row = x + size_t(i) * k;
            if (vec && j < k) {
                const float4 f = __ldg(reinterpret_cast<const float4 *>(row + j));
                v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) v[c] = j + c < k ? __ldg(row + j + c) : 0.f;
            }
        };
#pragma unroll
        for (int i = 0; i < M; ++i) {
            float most = 0.f;
            if (i < m)
#pragma unroll 4
                for (int j = 4 * threadIdx.x; j < pitch; j += 4 * kWarps * 32) {
                    float v[4];
                    load4(i, j, v);
                    most = katsu_larger4(most, v);
                }
            most = katsu_larger_of_warp(most);
            if (lane == 0) largest[i][warp] = most;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < M; ++i) {
            float most = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) most = katsu_larger(most, largest[i][w]);
            const KatsuInt8Scale s = katsu_int8_scale(most);
            if (threadIdx.x == 0) scales[i] = s.scale;
#pragma unroll 4
            for (int j = 4 * threadIdx.x; j < pitch; j += 4 * kWarps * 32) {
                float v[4] = {0.f, 0.f, 0.f, 0.f};
                if (i < m) load4(i, j, v);
                bool sure = true;
                unsigned out = katsu_int8_pack(v, s, &sure);
                if (!sure) out = katsu_int8_pack_exactly(v, s);
                *reinterpret_cast<unsigned *>(tokens + i * pitch + j) = out;
            }
        }
    } else {
        const int4 zero = make_int4(0, 0, 0, 0);
        for (int j = threadIdx.x; j < M * (pitch / 16); j += kWarps * 32)
            reinterpret_cast<int4 *>(tokens)[j] = j < m * (pitch / 16) ? __ldg(reinterpret_cast<const int4 *>(xq) + j) : zero;
        if (threadIdx.x < M) scales[threadIdx.x] = int(threadIdx.x) < m ? __ldg(xs + threadIdx.x) : 0.f;
    }
    __syncthreads();
    // ---- the weights ----
    bool fetched = true;
    for (int first = blockIdx.x * per_block; first < pairs; first += gridDim.x * per_block, fetched = false) {
        const int pair = first + warp / share;
        int acc[kRows][M] = {};
        if (pair < pairs) {
            for (int u0 = begin + lane; u0 - lane < end; u0 += 32 * kUnroll, fetched = false) {
                if (!fetched) fetch(pair, u0);
#pragma unroll
                for (int q = 0; q < kUnroll; ++q) {
                    if (u0 + 32 * q >= end) break;
#pragma unroll
                    for (int i = 0; i < M; ++i) {
                        const int4 t = *reinterpret_cast<const int4 *>(tokens + i * pitch + 16 * (u0 + 32 * q));
#pragma unroll
                        for (int r = 0; r < kRows; ++r) {
                            acc[r][i] = __dp4a(v[q][r].x, t.x, acc[r][i]);
                            acc[r][i] = __dp4a(v[q][r].y, t.y, acc[r][i]);
                            acc[r][i] = __dp4a(v[q][r].z, t.z, acc[r][i]);
                            acc[r][i] = __dp4a(v[q][r].w, t.w, acc[r][i]);
                        }
                    }
                }
            }
        }
        int mine = 0;  // result lane % (kRows * M) of the pair: row lane / M, token lane % M
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int i = 0; i < M; ++i) {
                const int s = __reduce_add_sync(0xffffffffu, acc[r][i]);
                if (lane == r * M + i) mine = s;
            }
        if (share > 1) {
            if (lane < kRows * M) sums[warp][lane] = mine;
            __syncthreads();
            if (part == 0 && lane < kRows * M)
                for (int p = 1; p < share; ++p) mine += sums[warp + p][lane];
        }
        const int row = pair * kRows + lane / M, token = lane % M;
        if (part == 0 && pair < pairs && lane < kRows * M && row < n && token < m)
            y[size_t(token) * n + row] = katsu_int8_result(mine, scales[token], __ldg(ws + row), bias ? __ldg(bias + row) : 0.f);
        if (share > 1) __syncthreads();
    }
}

}  // namespace

int32_t katsu_int8_few(katsu_cuda_ctx *ctx, const float *x, const int8_t *xq, const float *xs, const int8_t *wq,
                       const float *ws, const float *bias, float *y, size_t m, size_t k, size_t n, int *handled) {
    *handled = 0;
    const size_t pitch = katsu_int8_pitch(k);
    const int tokens = m <= 1 ? 1 : m <= 2 ? 2 : m <= 4 ? 4 : 8;
    const size_t smem = tokens * pitch;
    if (m > 8 || smem > kMostShared || n > 0x3fffffff) return KATSU_OK;
    // Rows in 8 bits come to every block as they are; rows in f32 are four times that, and read twice (2 x 8192 by 8192 x 8192:
    // 32 us, 19 with a launch that quantises them once).
    if (x != nullptr && m * k > 8192) return KATSU_OK;
    // Eight tokens' multiply-adds and their reads of shared memory take about as long as large weights: 8 x 8192 by 8192 x 8192
    // 27 us, on the tensor cores 22; 8 x 4096 by 4096 x 4096 8.5 and 10.5.
    if (m > 4 && k * n > (size_t(1) << 25)) return KATSU_OK;
    *handled = 1;
    auto kernel = tokens == 1 ? int8_rows_kernel<1> : tokens == 2 ? int8_rows_kernel<2> : tokens == 4 ? int8_rows_kernel<4> : int8_rows_kernel<8>;
    // Without asking, a block's tokens and the kernel's own variables (up to 800 bytes) have 48 KiB together.  All that a launch may
    // want is asked for once, so that none depends on the launches before it.
    KATSU_TRY(katsu_prepare_kernel(ctx, (const void *)kernel, kMostShared, false));
    const size_t pairs = katsu_div_up(n, kRows), warps = size_t(ctx->num_sms) * kWarps * 2;
    int share = 1;
    while (share < kWarps && pairs * share * 2 <= warps) share *= 2;
    const size_t need = katsu_div_up(pairs, kWarps / share);
    size_t fit = (size_t(224) * 1024) / (smem + 2048);  // blocks that an SM holds
    const size_t by_registers = tokens <= 2 ? 4 : 3;
    if (fit > by_registers) fit = by_registers;
    const size_t most = size_t(ctx->num_sms) * fit;
    return katsu_launch_chained(ctx, kernel, (unsigned)(need < most ? need : most), kWarps * 32, smem, 1, x, xq, xs, wq, ws, bias, y,
                                (int)m, (int)k, (int)n, (int)pitch, share);
}
