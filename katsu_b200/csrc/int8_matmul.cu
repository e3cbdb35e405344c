// y = (x in 8 bits) (w in 8 bits) with a scale for each token and channel: entry points, and the product for many tokens.
//
//   sum[channel][token] = sum_k  w_q[channel][k] x_q[token][k]      lanes channels (contiguous in y), columns tokens
//
// on tcgen05.mma kind::i8 (256 x bn x 32, 32-bit integer accumulators) on pairs of thread blocks.  Operands come by TMA as
// rows of 128 bytes; the epilogue multiplies a lane's sums with its channel's scale and each column's token scale, and a
// warp stores 128 contiguous bytes a column.  Integer sums are exact whatever their order, so an accumulator is read once, at
// the end of a tile, and a long k with few tiles is split over blocks whose sums a second launch adds up.
//
// Roles: warps 0-7 the epilogue (lane quarter = warp % 4, alternate 32-column chunks by warp / 4), warp 8 the TMA loads, warp
// 9 of the leader block the MMAs.  Two accumulators of 256 columns take turns, so the stores of a tile run under the next
// tile's products.  Every wait is bounded; both blocks of a pair reach the cluster barrier at the end.
#include "int8.cuh"
#include "sm100.cuh"
#include "sm100_pair.cuh"

using namespace sm100;

namespace {

constexpr int BM = 128, BK = 128;  // BK bytes (values) a k-block
constexpr int A_BYTES = BM * BK;
constexpr int MAX_STAGES = 8;
constexpr int THREADS = 320;
constexpr int RASTER_M = 16;
constexpr int SMEM_RING = 208 * 1024;
constexpr size_t SMEM = SMEM_RING + 1024;

struct Problem {
    float *y;
    int *partial;  // splits > 1: [splits][tokens][channels]
    const float *xs, *ws, *bias;
    int channels, tokens;
    int kblocks, last_steps;  // k-blocks of 128, steps of 32 in the last one
    int bn, m_tiles, n_tiles, splits, kb_per_split;
    int *status;
};

struct Maps {
    CUtensorMap w, x;
};

struct Tile {
    int split, mt, nt;
};

// Bands of RASTER_M tiles of channels, column-major inside a band: blocks running together share operand tiles in L2.
__device__ __forceinline__ Tile tile_of(int item, const Problem &p) {
    Tile t;
    const int per_split = p.m_tiles * p.n_tiles;
    t.split = item / per_split;
    const int i = item - t.split * per_split;
    const int band = i / (RASTER_M * p.n_tiles), r = i - band * (RASTER_M * p.n_tiles);
    const int rows = min(p.m_tiles - band * RASTER_M, RASTER_M);
    t.nt = r / rows;
    t.mt = band * RASTER_M + (r - t.nt * rows);
    return t;
}

// PER: k-blocks to a stage.  The issuing thread's waits and releases, once a stage, take about 470 clocks, in which the operands of two
// or four narrow blocks arrive and are multiplied (1024 x 4096 by 4096 x 512, tiles of 32 tokens: 12.1 us with one, 8.6 with four;
// by 4096 x 2048, tiles of 128: 13.3 with one, 10.7 with two).  Wider tiles would have three stages or fewer of more than one.
template <int PER>
__global__ void __launch_bounds__(THREADS, 1) int8_pair_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Problem p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int items = p.m_tiles * p.n_tiles * p.splits;
    const int half = p.bn >> 1;  // columns of B that this block loads
    const int b_bytes = half * BK, a_bytes = PER * A_BYTES, stage_bytes = PER * (A_BYTES + b_bytes);
    const int stages = min(MAX_STAGES, SMEM_RING / stage_bytes);
    launch_next();

    if (threadIdx.x == 0) {
        for (int s = 0; s < MAX_STAGES; ++s) {
            mbar_init(&full[s], 1);   // the leader's: its own expect_tx arrival, both blocks' bytes
            mbar_init(&empty[s], 1);  // each block's own copy, released by the leader's commit
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);    // each block's own copy
            mbar_init(&acc_empty[b], 16);  // the leader's: eight epilogue warps of each block
        }
        mbar_init_fence();
    }
    if (warp == 9) {
        tmem_alloc_pair(&tmem_slot, 512);
        tmem_relinquish_pair();
    }
    if (warp == 8 && lane < 2) tma_prefetch_desc(lane ? &maps.x : &maps.w);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();  // both blocks' barriers exist before anything is signalled across the pair
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_slot;
    launch_wait();

    if (warp == 8 && lane == 0) {
        bool ok = true;
        int s = 0;
        uint32_t phase = 1;  // a fresh barrier counts as released
        for (int item = pair; item < items && ok; item += pairs) {
            const Tile t = tile_of(item, p);
            const int m0 = (2 * t.mt + int(rank)) * BM, n0 = t.nt * p.bn + int(rank) * half;
            const int kb1 = min((t.split + 1) * p.kb_per_split, p.kblocks);
            for (int kb = t.split * p.kb_per_split; kb < kb1; kb += PER) {
                if (!mbar_wait(&empty[s], phase, p.status, 181)) { ok = false; break; }
                const int count = min(PER, kb1 - kb);
                if (leader) mbar_arrive_expect_tx(&full[s], 2 * count * (A_BYTES + b_bytes));
                const uint32_t bar = map_to_rank(&full[s], 0);
                unsigned char *st = smem + s * stage_bytes;
#pragma unroll
                for (int c = 0; c < PER; ++c) {
                    if (c >= count) break;
                    tma_load_3d_pair(st + c * A_BYTES, &maps.w, bar, (kb + c) * BK, m0, 0);
                    tma_load_3d_pair(st + a_bytes + c * b_bytes, &maps.x, bar, (kb + c) * BK, n0, 0);
                }
                if (++s == stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 9 && leader) {
        // whole warp in the loop, the elect.sync thread issues
        const bool issue = elect_one();
        const uint32_t idesc = idesc_i8(2 * BM, p.bn);
        bool ok = true;
        int s = 0, q = 0;  // q: accumulator hand-overs so far
        uint32_t phase = 0;
        for (int item = pair; item < items && ok; item += pairs, ++q) {
            const int split = item / (p.m_tiles * p.n_tiles);
            const int kb0 = split * p.kb_per_split, kb1 = min(kb0 + p.kb_per_split, p.kblocks);
            const int b = q & 1;
            if (!mbar_wait_warp_ready(&acc_empty[b], ((q >> 1) & 1) ^ 1, p.status, 182)) break;
            tc_fence_after_sync();
            const uint32_t acc = tmem_base + uint32_t(b * 256);
            for (int kb = kb0; kb < kb1; kb += PER) {
                if (!mbar_wait_warp_ready(&full[s], phase, p.status, 183)) { ok = false; break; }
                tc_fence_after_sync();
                const uint32_t st = smem_u32(smem + s * stage_bytes);
                const int count = min(PER, kb1 - kb);
                if (issue) {
#pragma unroll
                    for (int c = 0; c < PER; ++c) {
                        if (c >= count) break;
                        const uint64_t a0 = smem_desc(st + c * A_BYTES, 16, 1024, kLayoutSw128);
                        const uint64_t b0 = smem_desc(st + a_bytes + c * b_bytes, 16, 1024, kLayoutSw128);
                        const int steps = kb + c == p.kblocks - 1 ? p.last_steps : BK / 32;
#pragma unroll
                        for (int j = 0; j < BK / 32; ++j)
                            if (j < steps) mma_i8_pair(acc, a0 + j * 2, b0 + j * 2, idesc, kb + c > kb0 || j > 0);
                    }
                    // The accumulator's release comes last: the blocks leave when it has been drained, and no arrival may be
                    // outstanding then.
                    mma_commit_both(&empty[s]);
                    if (kb + count >= kb1) mma_commit_both(&acc_full[b]);
                }
                __syncwarp();
                if (++s == stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp < 8) {
        // thread = channel, alternate chunks of 32 tokens
        const int quarter = warp & 3, group = warp >> 2;
        int q = 0;
        for (int item = pair; item < items; item += pairs, ++q) {
            const Tile t = tile_of(item, p);
            const int channel = (2 * t.mt + int(rank)) * BM + quarter * 32 + lane, n0 = t.nt * p.bn, b = q & 1;
            const bool valid = channel < p.channels;
            const bool split = p.splits > 1;
            const float ws = valid && !split ? __ldg(p.ws + channel) : 0.f;
            const float bias = valid && !split && p.bias ? __ldg(p.bias + channel) : 0.f;
            if (!mbar_wait_warp(&acc_full[b], (q >> 1) & 1, p.status, 184)) break;
            tc_fence_after_sync();
            const uint32_t acc = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(b * 256);
            for (int c0 = group * 32; c0 < p.bn; c0 += 64) {
                const int token = n0 + c0, live = min(p.tokens - token, 32);
                if (live <= 0) break;
                const float scale = !split && lane < live ? __ldg(p.xs + token + lane) : 0.f;
                float v[32];
                tmem_ld_32x32(acc + c0, v);
                if (split) {
                    int *d = p.partial + (size_t(t.split) * p.tokens + token) * p.channels + channel;
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (valid && i < live) d[size_t(i) * p.channels] = __float_as_int(v[i]);
                } else {
                    float *d = p.y + size_t(token) * p.channels + channel;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float o = katsu_int8_result(__float_as_int(v[i]), __shfl_sync(0xffffffffu, scale, i), ws, bias);
                        if (valid && i < live) *d = o;
                        d += p.channels;
                    }
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (leader) mbar_arrive(&acc_empty[b]);
                else mbar_arrive_cluster(map_to_rank(&acc_empty[b], 0));
            }
        }
    }
    // Neither block leaves (or gives its tensor memory back) while the other may still signal its barriers, read its half of B
    // or hold accumulators: every path above ends here.
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    if (warp == 9) tmem_dealloc_pair(tmem_base, 512);
}

// y from the sums of all splits.
__global__ void __launch_bounds__(256) int8_fold_kernel(const int *__restrict__ partial, int splits, const float *__restrict__ xs,
                                                        const float *__restrict__ ws, const float *bias, float *y, size_t count,
                                                        unsigned channels) {
    launch_next();
    launch_wait();
    for (size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x; i < count; i += size_t(gridDim.x) * blockDim.x) {
        int sum = 0;
#pragma unroll 16
        for (int s = 0; s < splits; ++s) sum += __ldcg(partial + size_t(s) * count + i);
        const size_t token = i / channels;
        const unsigned channel = unsigned(i - token * channels);
        y[i] = katsu_int8_result(sum, __ldg(xs + token), __ldg(ws + channel), bias ? __ldg(bias + channel) : 0.f);
    }
}

int per_stage(int bn) { return bn <= 64 ? 4 : bn <= 160 ? 2 : 1; }

// Columns a tile and splits of k, by estimated clocks.  A k-block costs the tensor pipe 2 * bn, and the fill of (128 + bn / 2) * 128
// bytes a block at the rate of L2, 60 bytes a clock for each of 148 blocks and at most 75; a stage's waits are its least.  A tile's
// start is hidden but for the first one's, its stores but for the last one's (27 clocks a column where all blocks store at
// once); splits cost the writing and folding of their sums.
struct Plan {
    int bn, splits;
};
Plan plan_for(const katsu_cuda_ctx *ctx, size_t m, size_t k, size_t n) {
    const double pairs = ctx->num_sms / 2, results = double(m) * double(n);
    const long long kblocks = (long long)katsu_div_up(k, BK), m_tiles = (long long)katsu_div_up(n, 2 * BM);
    Plan best = {0, 1};
    double best_cost = 0;
    for (int bn = 32; bn <= 256; bn += 32) {
        const long long tiles = m_tiles * (long long)katsu_div_up(m, bn);
        const double pipe = 2.0 * bn, least = per_stage(bn) == 4 ? 285 : per_stage(bn) == 2 ? 300 : 470;
        for (int w = 0; w <= 2; ++w) {  // unsplit, or as many splits as fill one or two waves
            long long splits = w == 0 ? 1 : (long long)(w * pairs) / tiles;
            if (w > 0 && splits <= 1) continue;
            if (splits > kblocks / 2) splits = kblocks / 2;
            while (splits > 1 && splits * results > 6.4e7) --splits;  // 256 MB of sums
            if (splits < 1) splits = 1;
            const long long kb = (kblocks + splits - 1) / splits;
            splits = (kblocks + kb - 1) / kb;
            const double items = double(tiles * splits), waves = ceil(items / pairs), active = items < pairs ? items : pairs;
            const double rate = 60 * pairs / active, fill = (BM + bn / 2) * 128.0 / (rate < 75 ? rate : 75);
            const double busy = pipe > fill ? pipe : fill, per_kb = (busy > least ? busy : least) + 10;
            double cost = waves * (kb * per_kb + 200) + 1200 + bn * 27;
            if (splits > 1) cost += (splits + 1) * results * 4 / 2500 + 4000;
            if (best.bn == 0 || cost < best_cost) {
                best.bn = bn;
                best.splits = (int)splits;
                best_cost = cost;
            }
        }
    }
    return best;
}

bool rows_map(CUtensorMap *map, const int8_t *q, size_t rows, size_t pitch, int box_rows) {
    katsu_tensor_map_encode_fn encode = katsu_tensor_map_encoder();
    if (encode == nullptr) return false;
    cuuint64_t dims[3] = {pitch, rows, 1}, strides[2] = {pitch, pitch * rows};
    cuuint32_t box[3] = {BK, (cuuint32_t)box_rows, 1}, estr[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t *>(q), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// `partial`: plan.splits * m * n integers where the plan splits.
int32_t many(katsu_cuda_ctx *ctx, const Plan &plan, int *partial, const int8_t *xq, const float *xs, const int8_t *wq,
             const float *ws, const float *bias, float *y, size_t m, size_t k, size_t n) {
    const size_t pitch = katsu_int8_pitch(k);
    Maps maps;
    if (!rows_map(&maps.w, wq, n, pitch, BM) || !rows_map(&maps.x, xq, m, pitch, plan.bn / 2))
        return katsu_set_error(KATSU_ERR_CUDA, "cuTensorMapEncodeTiled failed for an 8-bit operand");
    Problem p = {};
    p.y = y;
    p.partial = partial;
    p.xs = xs; p.ws = ws; p.bias = bias;
    p.channels = (int)n;
    p.tokens = (int)m;
    p.kblocks = (int)katsu_div_up(pitch, BK);
    p.last_steps = (int)(katsu_div_up(pitch, 32) - 4 * (size_t(p.kblocks) - 1));
    p.bn = plan.bn;
    p.m_tiles = (int)katsu_div_up(n, 2 * BM);
    p.n_tiles = (int)katsu_div_up(m, plan.bn);
    p.splits = plan.splits;
    p.kb_per_split = (int)katsu_div_up(p.kblocks, plan.splits);
    p.status = ctx->status;
    const long long items = (long long)p.m_tiles * p.n_tiles * p.splits;
    if (items > 0x3fffffff) return katsu_set_error(KATSU_ERR_UNSUPPORTED, "too many tiles");
    const unsigned pairs = (unsigned)(items < ctx->num_sms / 2 ? items : ctx->num_sms / 2);
    auto kernel = per_stage(plan.bn) == 4 ? int8_pair_kernel<4> : per_stage(plan.bn) == 2 ? int8_pair_kernel<2> : int8_pair_kernel<1>;
    KATSU_TRY(katsu_prepare_kernel(ctx, (const void *)kernel, SMEM));
    KATSU_TRY(katsu_launch_chained(ctx, kernel, 2 * pairs, THREADS, SMEM, 2, maps, p));
    if (plan.splits == 1) return KATSU_OK;
    size_t blocks = katsu_div_up(m * n, 256);
    if (blocks > size_t(ctx->num_sms) * 8) blocks = size_t(ctx->num_sms) * 8;
    KATSU_TRY(katsu_prepare_kernel(ctx, (const void *)int8_fold_kernel, 0));
    return katsu_launch_chained(ctx, int8_fold_kernel, (unsigned)blocks, 256, 0, 1, partial, plan.splits, xs, ws, bias, y, m * n,
                                (unsigned)n);
}

int32_t check(const int8_t *wq, const float *ws, const float *y, size_t m, size_t k, size_t n) {
    KATSU_REQUIRE(k >= 1 && k <= KATSU_INT8_MAX_K, "k must be 1 to KATSU_INT8_MAX_K");
    KATSU_REQUIRE(m <= 0x3fffffff && n <= 0x3fffffff, "too many rows or columns");
    if (m == 0 || n == 0) return KATSU_OK;
    KATSU_REQUIRE(wq != nullptr && ws != nullptr && y != nullptr, "null buffer");
    KATSU_REQUIRE((reinterpret_cast<uintptr_t>(wq) & 15u) == 0, "a quantised matrix must be 16-byte aligned");
    return KATSU_OK;
}

// x: `x_bytes` of tokens, in 8 bits with scales xs or in f32.
int32_t check_apart(const float *y, const void *x, size_t x_bytes, const float *xs, const int8_t *wq, const float *ws,
                    const float *bias, size_t m, size_t k, size_t n) {
    const size_t bytes = m * n * sizeof(float), channels = n * sizeof(float);
    const bool apart = !katsu_overlap(y, bytes, x, x_bytes) && !katsu_overlap(y, bytes, xs, m * sizeof(float)) &&
                       !katsu_overlap(y, bytes, wq, n * katsu_int8_pitch(k)) && !katsu_overlap(y, bytes, ws, channels) &&
                       !katsu_overlap(y, bytes, bias, channels);
    KATSU_REQUIRE(apart, "y is an input too, or overlaps one");
    return KATSU_OK;
}

}  // namespace

extern "C" int32_t katsu_cuda_int8_matmul(katsu_cuda_ctx *ctx, const int8_t *xq, const float *xs, const int8_t *wq,
                                          const float *ws, const float *bias, float *y, size_t m, size_t k, size_t n) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_TRY(check(wq, ws, y, m, k, n));
    if (m == 0 || n == 0) return katsu_bind(ctx);
    KATSU_REQUIRE(xq != nullptr && xs != nullptr, "null buffer");
    KATSU_TRY(check_apart(y, xq, m * katsu_int8_pitch(k), xs, wq, ws, bias, m, k, n));
    KATSU_REQUIRE((reinterpret_cast<uintptr_t>(xq) & 15u) == 0, "a quantised matrix must be 16-byte aligned");
    KATSU_TRY(katsu_bind(ctx));
    int handled = 0;
    KATSU_TRY(katsu_int8_few(ctx, nullptr, xq, xs, wq, ws, bias, y, m, k, n, &handled));
    if (handled) return KATSU_OK;
    const Plan plan = plan_for(ctx, m, k, n);
    float *scratch = nullptr;
    if (plan.splits > 1) KATSU_TRY(katsu_scratch(ctx, size_t(plan.splits) * m * n, &scratch));
    return many(ctx, plan, reinterpret_cast<int *>(scratch), xq, xs, wq, ws, bias, y, m, k, n);
}

extern "C" int32_t katsu_cuda_int8_linear(katsu_cuda_ctx *ctx, const float *x, const int8_t *wq, const float *ws,
                                          const float *bias, float *y, size_t m, size_t k, size_t n) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_TRY(check(wq, ws, y, m, k, n));
    if (m == 0 || n == 0) return katsu_bind(ctx);
    KATSU_REQUIRE(x != nullptr, "null buffer");
    KATSU_TRY(check_apart(y, x, m * k * sizeof(float), nullptr, wq, ws, bias, m, k, n));
    KATSU_TRY(katsu_bind(ctx));
    int handled = 0;
    KATSU_TRY(katsu_int8_few(ctx, x, nullptr, nullptr, wq, ws, bias, y, m, k, n, &handled));
    if (handled) return KATSU_OK;
    const Plan plan = plan_for(ctx, m, k, n);
    // x in 8 bits, its scales and, where k is split, the sums of its parts
    const size_t xq_floats = katsu_div_up(m * katsu_int8_pitch(k), 256) * 64, scales = katsu_div_up(m, 64) * 64;
    float *scratch = nullptr;
    KATSU_TRY(katsu_scratch(ctx, xq_floats + scales + (plan.splits > 1 ? size_t(plan.splits) * m * n : 0), &scratch));
    int8_t *xq = reinterpret_cast<int8_t *>(scratch);
    float *xs = scratch + xq_floats;
    KATSU_TRY(katsu_int8_quantize(ctx, x, xq, xs, m, k));
    KATSU_TRY(katsu_int8_few(ctx, nullptr, xq, xs, wq, ws, bias, y, m, k, n, &handled));
    if (handled) return KATSU_OK;
    return many(ctx, plan, reinterpret_cast<int *>(xs + scales), xq, xs, wq, ws, bias, y, m, k, n);
}
