// Matrices to 8 bits: rows of x (one scale a token) and columns of w (one scale an output channel, kept transposed).
//
// Rows: a warp (up to 1024 values), a block of 128 to 1024 threads or a cluster of blocks takes a row and holds it in registers, 32
// values a thread, between the largest magnitude and the quotients; of rows that a block cannot hold what lies in front of
// these is read again, from L2.  Bound: HBM, 4 bytes in and 1 out a value (8192 x 8192: 53 us, its floor 52).
//
// Columns: one launch finds the largest magnitudes of pieces of the columns, another folds them and turns tiles of 128 x 32 over
// in shared memory; w is read twice, the second time from L2 where it fits.
#include "int8.cuh"
#include "sm100_pair.cuh"

using namespace sm100;

namespace {

// Values j .. j + 3 of a row, zeros behind its end.
template <bool VEC>
__device__ __forceinline__ void load4(const float *row, size_t j, size_t k, float (&v)[4]) {
    if (VEC && j + 4 <= k) {
        const float4 f = __ldg(reinterpret_cast<const float4 *>(row + j));
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = j + i < k ? __ldg(row + j + i) : 0.f;
    }
}

constexpr int kHeld = 8;        // 16-byte pieces
constexpr int kMostBlocks = 8;  // to a row: 131072 values are held

// C blocks of T threads to a row, each thread with kHeld 16-byte pieces: the row's last ones, loaded behind what is read twice, so
// that their registers are free until then.  WAVES: more blocks than are resident at once (see katsu_int8_quantize).
template <int T, int C, bool VEC, bool WAVES>
__global__ void __launch_bounds__(T == 32 ? 256 : T, WAVES && T < 512 ? 1 : T == 32 ? 3 : 1024 / T)
quantize_rows_kernel(const float *__restrict__ x, int8_t *q, float *scale, unsigned long long rows, size_t k, size_t pitch) {
    __shared__ float sh[T / 32], of_block;
    if (!WAVES) launch_next();
    launch_wait();
    constexpr int per_block = T == 32 ? 8 : 1, TC = T * C, batch = 4 * TC * kHeld;
    const int t = threadIdx.x % T + (C > 1 ? int(cluster_ctarank()) * T : 0);
    const unsigned long long row = C > 1 ? blockIdx.x / C : (unsigned long long)blockIdx.x * per_block + threadIdx.x / T;
    if (row >= rows) return;  // (a warp's rows: the others of the block do not wait)
    const float *src = x + row * k;
    const size_t twice = T == 1024 || C == kMostBlocks ? (pitch - 1) / batch * batch : 0;  // values in front of the held ones
    float most = 0.f;
    for (size_t j0 = 0; j0 < twice; j0 += batch) {
        float v[kHeld][4];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) load4<VEC>(src, j0 + 4 * (t + i * TC), k, v[i]);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) most = katsu_larger4(most, v[i]);
    }
    float v[kHeld][4];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) load4<VEC>(src, twice + 4 * (t + i * TC), k, v[i]);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) most = katsu_larger4(most, v[i]);
    most = katsu_larger_of_warp(most);
    if (T > 32) {
        if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < T / 32; ++w) most = katsu_larger(most, sh[w]);
    }
    if (C > 1) {
        if (threadIdx.x == 0) of_block = most;
        __syncwarp();
        cluster_sync_all();
#pragma unroll
        for (int c = 0; c < C; ++c) most = katsu_larger(most, ld_cluster(map_to_rank(&of_block, c)));
        cluster_arrive();  // (a block leaves when the others have read what it found)
    }
    const KatsuInt8Scale s = katsu_int8_scale(most);
    if (t == 0) scale[row] = s.scale;
    unsigned *dst = reinterpret_cast<unsigned *>(q + row * pitch);
    bool sure = true;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const size_t j = twice + 4 * (t + i * TC);
        const unsigned out = katsu_int8_pack(v[i], s, &sure);
        if (j < pitch) dst[j / 4] = out;
    }
    for (size_t j0 = 0; j0 < twice; j0 += batch) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) load4<VEC>(src, j0 + 4 * (t + i * TC), k, v[i]);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) dst[(j0 + 4 * (t + i * TC)) / 4] = katsu_int8_pack(v[i], s, &sure);
    }
    if (!sure)  // this thread's pieces once more, by the definition
        for (size_t j = 4 * t; j < pitch; j += 4 * TC) {
            float w[4];
            load4<VEC>(src, j, k, w);
            dst[j / 4] = katsu_int8_pack_exactly(w, s);
        }
    if (C > 1) {
        __syncwarp();
        cluster_wait();
    }
}

// Largest magnitude of every column of w [k, n] over each of `pieces` equal pieces of its rows: [pieces][n].  A block has a piece
// of 32 columns.
__global__ void __launch_bounds__(256) column_largest_kernel(const float *__restrict__ w, float *largest, size_t k, size_t n,
                                                             unsigned pieces, unsigned tiles, int waves) {
    if (!waves) launch_next();
    launch_wait();
    const unsigned piece = blockIdx.x / tiles, lane = threadIdx.x & 31;
    const size_t col = size_t(blockIdx.x - piece * tiles) * 32 + lane;
    const size_t begin = k * piece / pieces, end = k * (piece + 1) / pieces;
    float m = 0.f;
    if (col < n)
#pragma unroll 8
        for (size_t p = begin + (threadIdx.x >> 5); p < end; p += 8) m = katsu_larger(m, __ldg(w + p * n + col));
    __shared__ float sh[8][33];
    sh[threadIdx.x >> 5][lane] = m;
    __syncthreads();
    if (threadIdx.x < 32 && col < n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m = katsu_larger(m, sh[i][lane]);
        largest[piece * n + col] = m;
    }
}

constexpr int kTileBlocks = 5;  // of the kernel below that an SM holds at once

// A tile of 128 rows of w by 32 columns to 32 rows of q.  A thread has 16 rows of one column, so that it needs one scale (with tiles
// turned over in f32 and a scale for each of a thread's four columns: 30 us at 4096 x 4096, now 20), and four of their whole
// numbers are a word of the tile that shared memory turns over.
__global__ void __launch_bounds__(256, kTileBlocks) quantize_columns_kernel(const float *__restrict__ w, const float *largest, int8_t *q,
                                                                            float *scale, size_t k, size_t n, size_t pitch,
                                                                            unsigned pieces, unsigned tiles, int waves) {
    __shared__ unsigned tile[32][33];  // [column][word]
    __shared__ float sh[8][32];
    if (!waves) launch_next();
    launch_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned part = blockIdx.x / tiles;
    const size_t p0 = size_t(part) * 128, col0 = size_t(blockIdx.x - part * tiles) * 32;
    const bool in = col0 + lane < n;
    const float *src = w + (p0 + 16 * warp) * n + col0 + lane;
    float v[4][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        v[i >> 2][i & 3] = in && p0 + 16 * warp + i < k ? __ldg(src) : 0.f;
        src += n;
    }
    float m = 0.f;
    if (in)
        for (unsigned piece = warp; piece < pieces; piece += 8) m = katsu_larger(m, __ldcg(largest + piece * n + col0 + lane));
    sh[warp][lane] = m;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) m = katsu_larger(m, sh[j][lane]);
    const KatsuInt8Scale s = katsu_int8_scale(m);
    if (part == 0 && warp == 0 && in) scale[col0 + lane] = s.scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bool sure = true;
        unsigned out = katsu_int8_pack(v[i], s, &sure);
        if (!sure) out = katsu_int8_pack_exactly(v[i], s);
        tile[lane][4 * warp + i] = out;
    }
    __syncthreads();
    const size_t p = p0 + 4 * lane;
    if (p >= pitch) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const size_t col = col0 + warp + 8 * i;
        if (col < n) *reinterpret_cast<unsigned *>(q + col * pitch + p) = tile[warp + 8 * i][lane];
    }
}

}  // namespace

template <bool VEC, bool WAVES>
static void (*rows_kernel(size_t k, unsigned cluster))(const float *, int8_t *, float *, unsigned long long, size_t, size_t) {
    return cluster == 2   ? quantize_rows_kernel<512, 2, VEC, WAVES>
           : cluster == 4 ? quantize_rows_kernel<512, 4, VEC, WAVES>
           : cluster > 4  ? quantize_rows_kernel<512, kMostBlocks, VEC, WAVES>
           : k <= 1024    ? quantize_rows_kernel<32, 1, VEC, WAVES>
           : k <= 4096    ? quantize_rows_kernel<128, 1, VEC, WAVES>
           : k <= 8192    ? quantize_rows_kernel<256, 1, VEC, WAVES>
           : k <= 16384   ? quantize_rows_kernel<512, 1, VEC, WAVES> : quantize_rows_kernel<1024, 1, VEC, true>;
}

// A row to a warp or block.  Few rows: the launch is chained, like that of the product behind it.  More rows than go round at once:
// the hardware hands them out as others end, and the rounds of one hide behind the loads of others.  Either way the kernel wants
// its L1 for the loads in flight (8192 x 8192: 53 us, with the largest shared-memory partition 80; 64 x 8192 3.1 and 4.3).
//
// Rows of more than 16384 values: clusters of blocks hold each of them where about all are resident at once (with the product,
// 30 rows of 65536: 16 us, a block to a row 19).  Else clusters wait for places in one group of SMs and a block to a row is
// faster, that reads what it cannot hold twice (512 rows of 65536: 54 us, in clusters 57).
int32_t katsu_int8_quantize(katsu_cuda_ctx *ctx, const float *x, int8_t *q, float *scale, size_t m, size_t k) {
    const bool vec = k % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
    const bool warps = k <= 1024;
    const size_t sms = ctx->num_sms;
    unsigned threads = warps ? 256 : k <= 4096 ? 128 : k <= 8192 ? 256 : 512, cluster = 1;
    if (k > 16384) {
        cluster = k <= 32768 ? 2 : k <= 65536 ? 4 : kMostBlocks;
        if (m * cluster > sms * 2) {
            cluster = 1;
            threads = 1024;
        }
    }
    const size_t blocks = warps ? katsu_div_up(m, 8) : m * cluster;
    // (as the kernels' bounds; clusters leave some SMs idle)
    const bool waves = blocks > sms * (warps ? 3 : cluster > 1 ? 1 : 1024 / threads);
    auto kernel = waves ? (vec ? rows_kernel<true, true>(k, cluster) : rows_kernel<false, true>(k, cluster))
                        : (vec ? rows_kernel<true, false>(k, cluster) : rows_kernel<false, false>(k, cluster));
    return katsu_launch(ctx, !waves, kernel, (unsigned)blocks, threads, 0, cluster, x, q, scale, m, k, katsu_int8_pitch(k));
}

extern "C" int32_t katsu_cuda_int8_row_bytes(size_t k, size_t *out_bytes) {
    KATSU_REQUIRE(out_bytes != nullptr, "out_bytes is null");
    KATSU_REQUIRE(k >= 1 && k <= KATSU_INT8_MAX_K, "k must be 1 to KATSU_INT8_MAX_K");
    *out_bytes = katsu_int8_pitch(k);
    return KATSU_OK;
}

// `rows` rows of k values to 8 bits.
static int32_t check_apart(const float *v, const int8_t *q, const float *scale, size_t rows, size_t k) {
    const size_t in = rows * k * sizeof(float), out = rows * katsu_int8_pitch(k), scales = rows * sizeof(float);
    const bool apart = !katsu_overlap(q, out, v, in) && !katsu_overlap(scale, scales, v, in) && !katsu_overlap(q, out, scale, scales);
    KATSU_REQUIRE(apart, "the input and the outputs overlap");
    return KATSU_OK;
}

extern "C" int32_t katsu_cuda_int8_quantize_rows(katsu_cuda_ctx *ctx, const float *x, int8_t *q, float *scale, size_t m,
                                                 size_t k) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_REQUIRE(k >= 1 && k <= KATSU_INT8_MAX_K, "k must be 1 to KATSU_INT8_MAX_K");
    KATSU_REQUIRE(m <= 0x7fffffff, "too many rows");
    if (m == 0) return katsu_bind(ctx);
    KATSU_REQUIRE(x != nullptr && q != nullptr && scale != nullptr, "null buffer");
    KATSU_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15u) == 0, "a quantised matrix must be 16-byte aligned");
    KATSU_TRY(check_apart(x, q, scale, m, k));
    KATSU_TRY(katsu_bind(ctx));
    return katsu_int8_quantize(ctx, x, q, scale, m, k);
}

extern "C" int32_t katsu_cuda_int8_quantize_weights(katsu_cuda_ctx *ctx, const float *w, int8_t *q, float *scale, size_t k,
                                                    size_t n) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_REQUIRE(k >= 1 && k <= KATSU_INT8_MAX_K, "k must be 1 to KATSU_INT8_MAX_K");
    KATSU_REQUIRE(n <= 0x7fffffff, "too many columns");
    if (n == 0) return katsu_bind(ctx);
    KATSU_REQUIRE(w != nullptr && q != nullptr && scale != nullptr, "null buffer");
    KATSU_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15u) == 0, "a quantised matrix must be 16-byte aligned");
    KATSU_TRY(check_apart(w, q, scale, n, k));
    KATSU_TRY(katsu_bind(ctx));
    const size_t tiles = katsu_div_up(n, 32), parts = katsu_div_up(k, 128), resident = size_t(ctx->num_sms) * 8;
    // pieces of at least 64 rows, about eight blocks to an SM
    size_t pieces = resident / tiles;
    if (pieces > katsu_div_up(k, 64)) pieces = katsu_div_up(k, 64);
    if (pieces < 1) pieces = 1;
    if (parts * tiles > 0x7fffffff) return katsu_set_error(KATSU_ERR_UNSUPPORTED, "too many weights");
    float *largest = nullptr;
    KATSU_TRY(katsu_scratch(ctx, pieces * n, &largest));
    const bool waves_a = pieces * tiles > resident, waves_b = parts * tiles > size_t(ctx->num_sms) * kTileBlocks;
    KATSU_TRY(katsu_launch(ctx, !waves_a, column_largest_kernel, (unsigned)(pieces * tiles), 256, 0, 1, w, largest, k, n,
                           (unsigned)pieces, (unsigned)tiles, waves_a ? 1 : 0));
    KATSU_TRY(katsu_launch(ctx, !waves_b, quantize_columns_kernel, (unsigned)(parts * tiles), 256, 0, 1, w, largest, q, scale, k, n,
                           katsu_int8_pitch(k), (unsigned)pieces, (unsigned)tiles, waves_b ? 1 : 0));
    return KATSU_OK;
}
