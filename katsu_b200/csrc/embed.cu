// Rows of a table for a list of tokens, and the gradient of the table.
//
//   y[i] = scale * table[t_i]                        dtable[v] (+)= scale * sum over i with t_i = v of dy[i]
//
// The lookup reads the rows of the tokens and writes y: HBM.  The gradient sorts the tokens (positions of one token in
// ascending order behind each other), cuts the sorted list into pieces of kPiece and adds up each piece on its own, whatever
// the tokens are: a token of a tenth of all positions costs what a thousand rare ones cost.  Runs that lie in one piece are
// written as they end; what a piece has of a run that began in front of it or goes on behind it is kept beside the table
// and folded by a second launch in the pieces' order.  No floating-point atomics: the same tokens give the same bits.
#include <algorithm>

#include "common.cuh"
#include "launch.cuh"

namespace {

constexpr int kThreads = 256;

template <int VEC>
struct Values {
    float v[VEC];
};

template <int VEC>
__device__ __forceinline__ Values<VEC> load(const float *p) {
    Values<VEC> r;
    if constexpr (VEC == 4) {
        const float4 f = *reinterpret_cast<const float4 *>(p);
        r.v[0] = f.x, r.v[1] = f.y, r.v[2] = f.z, r.v[3] = f.w;
    } else {
        r.v[0] = *p;
    }
    return r;
}

template <int VEC>
__device__ __forceinline__ void store(float *p, const Values<VEC> &r) {
    if constexpr (VEC == 4) *reinterpret_cast<float4 *>(p) = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
    else *p = r.v[0];
}

// ---- lookup ----------------------------------------------------------------------------------------------------------
// A row is `units` accesses of VEC values; 1 << shift threads share a row (a block's slab of 4 << shift accesses of it, where
// it is longer).  Four accesses of a thread are on their way together.
struct Rows {
    unsigned count, units, slabs;
    int shift;
};

Rows rows_of(size_t count, size_t units) {
    Rows r;
    r.count = unsigned(count);
    r.units = unsigned(units);
    r.shift = 0;
    while (r.shift < 8 && (size_t(1) << r.shift) < units) ++r.shift;
    r.slabs = unsigned(katsu_div_up(units, size_t(4) << r.shift));
    return r;
}

// INT8: the table's rows are int8_t of `pitch` bytes with a scale each, four values a load.
template <int VEC, bool INT8>
__global__ void __launch_bounds__(kThreads) embed_kernel(const void *table, const float *rows_scale, const int *tokens, float scale,
                                                         float *y, Rows rows, unsigned vocab, size_t pitch, size_t cols, int waves) {
    if (!waves) launch_next();
    launch_wait();
    const unsigned group = blockIdx.x / rows.slabs, slab = blockIdx.x % rows.slabs, width = 1u << rows.shift;
    const unsigned long long i = (unsigned long long)group * (kThreads >> rows.shift) + (threadIdx.x >> rows.shift);
    if (i >= rows.count) return;
    const unsigned token = unsigned(tokens[i]);
    const bool there = token < vocab;
    const unsigned u0 = slab * 4 * width + (threadIdx.x & (width - 1));
    float of_row = scale;
    if (INT8 && there) of_row = rows_scale[token];
    Values<VEC> v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const unsigned u = u0 + q * width;
#pragma unroll
        for (int c = 0; c < VEC; ++c) v[q].v[c] = 0.f;
        if (u >= rows.units || !there) continue;
        if constexpr (INT8) {
            const int8_t *row = static_cast<const int8_t *>(table) + size_t(token) * pitch;
            if constexpr (VEC == 4) {
                const char4 b = *reinterpret_cast<const char4 *>(row + 4 * size_t(u));
                v[q].v[0] = b.x, v[q].v[1] = b.y, v[q].v[2] = b.z, v[q].v[3] = b.w;
            } else {
                v[q].v[0] = row[u];
            }
        } else {
            v[q] = load<VEC>(static_cast<const float *>(table) + size_t(token) * cols + size_t(u) * VEC);
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const unsigned u = u0 + q * width;
        if (u >= rows.units) continue;
#pragma unroll
        for (int c = 0; c < VEC; ++c) v[q].v[c] = !there ? 0.f : INT8 ? (v[q].v[c] * of_row) * scale : v[q].v[c] * scale;
        store<VEC>(y + i * cols + size_t(u) * VEC, v[q]);
    }
}

bool vectors(const void *p, size_t cols) { return cols % 4 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int VEC, bool INT8>
int32_t launch_lookup(katsu_cuda_ctx *ctx, const void *table, const float *rows_scale, const int *tokens, float scale, float *y,
                      size_t count, size_t vocab, size_t pitch, size_t cols) {
    const Rows rows = rows_of(count, cols / VEC);
    const size_t blocks = katsu_div_up(count, kThreads >> rows.shift) * rows.slabs;
    if (blocks > 0x7fffffffu) return katsu_set_error(KATSU_ERR_UNSUPPORTED, "%zu rows of %zu values in one lookup", count, cols);
    const bool waves = blocks > size_t(2) * ctx->num_sms;
    return katsu_launch(ctx, !waves, embed_kernel<VEC, INT8>, unsigned(blocks), kThreads, 0, 1, table, rows_scale, tokens, scale, y, rows,
                        unsigned(vocab), pitch, cols, int(waves));
}

// ---- sorting the tokens --------------------------------------------------------------------------------------------------
// keys[p] and position[p]: the tokens in ascending order, equal ones by position, what is no token (key `vocab`) last.
constexpr int kRanked = 32, kMostRanked = 8192;

__device__ __forceinline__ unsigned key_of(int token, unsigned vocab) { return min(unsigned(token), vocab); }

// Up to 8192 tokens: the place of a token is the number of tokens that belong in front of it.  A block counts for 32 of them,
// its warps over an eighth of the list each: 64 comparisons a lane and cycle of the GPU, one launch (8192 tokens: 67 million
// comparisons).
__global__ void __launch_bounds__(256) rank_kernel(const int *tokens, unsigned count, unsigned vocab, unsigned *keys, int *position) {
    __shared__ __align__(16) unsigned all[kMostRanked];
    __shared__ int partial[8][kRanked];
    launch_next();
    launch_wait();
    const unsigned tiles = (count + 31) / 32, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (unsigned j = threadIdx.x; j < tiles * 32; j += 256) all[j] = j < count ? key_of(tokens[j], vocab) : 0xffffffffu;
    __syncthreads();
    const unsigned i = blockIdx.x * kRanked + lane, key = all[i];
    int before = 0;
    for (unsigned tile = warp; tile < tiles; tile += 8) {
        const uint4 *of_tile = reinterpret_cast<const uint4 *>(all + 32 * tile);
        const unsigned limit = key + (tile < blockIdx.x ? 1 : 0);  // in front: equal ones count too
#pragma unroll
        for (unsigned q = 0; q < 8; ++q) {
            const uint4 k = of_tile[q];
            before += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
        }
        if (tile == blockIdx.x)
            for (unsigned j = 0; j < lane; ++j) before += all[32 * tile + j] == key;
    }
    partial[warp][lane] = before;
    __syncthreads();
    if (warp != 0 || i >= count) return;
    int place = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) place += partial[w][lane];
    keys[place] = key;
    position[place] = int(i);
}

// More: passes over digits of up to 10 bits from the lowest on, two launches each.  A block has `tile` of the keys.
constexpr int kDigits = 1024, kSorters = 128;

struct Pass {
    const int *tokens;                              // first pass
    const unsigned *keys;                           // later ones
    const int *position;
    unsigned count, vocab, tile;
    int shift, bits;
};

__device__ __forceinline__ unsigned pass_key(const Pass &p, unsigned i) { return p.tokens ? key_of(p.tokens[i], p.vocab) : p.keys[i]; }

// digits[block][digit]: how many of the block's keys have the digit.
__global__ void __launch_bounds__(256) digits_kernel(Pass p, unsigned *digits) {
    __shared__ unsigned mine[kDigits];
    launch_next();
    const unsigned values = 1u << p.bits, mask = values - 1;
    for (unsigned d = threadIdx.x; d < values; d += 256) mine[d] = 0;
    __syncthreads();
    launch_wait();
    const unsigned begin = blockIdx.x * p.tile, end = min(p.count, begin + p.tile);
    for (unsigned i = begin + threadIdx.x; i < end; i += 256) atomicAdd(&mine[(pass_key(p, i) >> p.shift) & mask], 1u);
    __syncthreads();
    for (unsigned d = threadIdx.x; d < values; d += 256) digits[blockIdx.x * values + d] = mine[d];
}

// Moves the block's keys to their places.  A warp takes an eighth of them in order, so that equal digits keep theirs.
__global__ void __launch_bounds__(256) scatter_kernel(Pass p, const unsigned *digits, unsigned *keys, int *position) {
    __shared__ unsigned place[8][kDigits];
    __shared__ unsigned sums[8];
    launch_next();
    launch_wait();
    const unsigned values = 1u << p.bits, mask = values - 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (unsigned d = threadIdx.x; d < 8 * kDigits; d += 256) (&place[0][0])[d] = 0;
    __syncthreads();
    const unsigned share = p.tile / 8, begin = min(p.count, blockIdx.x * p.tile + warp * share), end = min(p.count, begin + share);
    for (unsigned i = begin + lane; i < end; i += 32) atomicAdd(&place[warp][(pass_key(p, i) >> p.shift) & mask], 1u);
    __syncthreads();
    // a thread's four digits: keys of each in all blocks and in those in front of this one
    unsigned all[4] = {0, 0, 0, 0}, front[4] = {0, 0, 0, 0};
    const unsigned d0 = 4 * threadIdx.x;
    if (d0 < values) {
#pragma unroll 8
        for (unsigned b = 0; b < gridDim.x; ++b) {
            const unsigned *of_block = digits + size_t(b) * values + d0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const unsigned n = d0 + q < values ? of_block[q] : 0;
                all[q] += n;
                front[q] += b < blockIdx.x ? n : 0;
            }
        }
    }
    unsigned sum = all[0] + all[1] + all[2] + all[3], scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned other = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= unsigned(o)) scan += other;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    unsigned first = scan - sum;
    for (unsigned w = 0; w < warp; ++w) first += sums[w];
    if (d0 < values) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            unsigned at = first + front[q];
            if (d0 + q < values)
                for (int w = 0; w < 8; ++w) {
                    const unsigned n = place[w][d0 + q];
                    place[w][d0 + q] = at;
                    at += n;
                }
            first += all[q];
        }
    }
    __syncthreads();
    for (unsigned i0 = begin; i0 < end; i0 += 32) {
        const unsigned i = i0 + lane;
        const bool valid = i < end;
        const unsigned key = valid ? pass_key(p, i) : 0, digit = valid ? (key >> p.shift) & mask : 0xffffffffu;
        const unsigned same = __match_any_sync(0xffffffffu, digit), ahead = __popc(same & ((1u << lane) - 1));
        unsigned at = 0;
        if (valid) at = place[warp][digit] + ahead;
        __syncwarp();
        if (valid && ahead == 0) place[warp][digit] += __popc(same);
        __syncwarp();
        if (!valid) continue;
        keys[at] = key;
        position[at] = p.tokens ? int(i) : p.position[i];
    }
}

// ---- the gradient ----------------------------------------------------------------------------------------------------------
constexpr int kPiece = 32, kGradThreads = 128;

struct Grad {
    const unsigned *keys;
    const int *position;
    const float *dy;
    float *dtable, *kept;  // kept [piece][2][pitch]: of the run that began in front; of the one that goes on behind
    float scale;
    unsigned count, vocab, units, slabs, pieces, piece_blocks, fill_rows;
    int shift, accumulate;
    size_t cols, pitch;
};

// First place of the sorted keys that is not below `key`.
__device__ __forceinline__ unsigned lower_bound(const unsigned *keys, unsigned count, unsigned key) {
    unsigned lo = 0, hi = count;
    while (lo < hi) {
        const unsigned mid = (lo + hi) >> 1;
        if (keys[mid] < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <int VEC>
__device__ __forceinline__ void write_row(const Grad &g, unsigned key, unsigned u, Values<VEC> sum) {
    float *dst = g.dtable + size_t(key) * g.cols + size_t(u) * VEC;
    Values<VEC> old;
    if (g.accumulate) old = load<VEC>(dst);
#pragma unroll
    for (int c = 0; c < VEC; ++c) sum.v[c] = g.accumulate ? fmaf(g.scale, sum.v[c], old.v[c]) : g.scale * sum.v[c];
    store<VEC>(dst, sum);
}

// Blocks 0 .. piece_blocks - 1: a group of 1 << shift threads adds up a piece (a slab of 1 << shift accesses of its rows); the
// blocks behind them write zeros to fill_rows rows of the table each, but for those of tokens that are there.
template <int VEC>
__global__ void __launch_bounds__(kGradThreads) embed_grad_kernel(Grad g) {
    const unsigned width = 1u << g.shift, groups = kGradThreads >> g.shift, mine = threadIdx.x >> g.shift, lane = threadIdx.x & (width - 1);
    __shared__ unsigned keys[kGradThreads / 4 * kPiece + 2];
    __shared__ int position[kGradThreads / 4 * kPiece];
    __shared__ bool there[kGradThreads];
    if (blockIdx.x >= g.piece_blocks) {
        const unsigned row0 = (blockIdx.x - g.piece_blocks) * g.fill_rows, rows = min(g.fill_rows, g.vocab - row0);
        if (threadIdx.x < rows) {
            const unsigned key = row0 + threadIdx.x, at = lower_bound(g.keys, g.count, key);
            there[threadIdx.x] = at < g.count && g.keys[at] == key;
        }
        __syncthreads();
        Values<VEC> zero;
#pragma unroll
        for (int c = 0; c < VEC; ++c) zero.v[c] = 0.f;
        for (unsigned r = mine; r < rows; r += groups) {
            if (there[r]) continue;
            float *row = g.dtable + size_t(row0 + r) * g.cols;
            for (unsigned u = lane; u < g.units; u += width) store<VEC>(row + size_t(u) * VEC, zero);
        }
        return;
    }
    const unsigned slab = blockIdx.x % g.slabs, piece0 = blockIdx.x / g.slabs * groups, begin0 = piece0 * kPiece;
    const unsigned staged = min(groups * kPiece, g.count - begin0);
    // keys[1 + j] is that of place begin0 + j; one in front and one behind as well, ~0 where there is none
    for (unsigned j = threadIdx.x; j < staged; j += kGradThreads) {
        keys[1 + j] = g.keys[begin0 + j];
        position[j] = g.position[begin0 + j];
    }
    if (threadIdx.x == 0) keys[0] = begin0 ? g.keys[begin0 - 1] : ~0u;
    if (threadIdx.x == 1) keys[1 + staged] = begin0 + staged < g.count ? g.keys[begin0 + staged] : ~0u;
    __syncthreads();
    const unsigned piece = piece0 + mine, u = slab * width + lane, j0 = mine * kPiece;
    if (piece >= g.pieces || u >= g.units) return;
    const unsigned j1 = min(staged, j0 + kPiece);
    float *kept = g.kept + size_t(piece) * 2 * g.pitch + size_t(u) * VEC;
    bool began = keys[j0] != keys[j0 + 1];  // the current run began in this piece
    Values<VEC> sum;
#pragma unroll
    for (int c = 0; c < VEC; ++c) sum.v[c] = 0.f;
    for (unsigned j = j0; j < j1; j += 8) {
        Values<VEC> v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (j + q < j1) v[q] = load<VEC>(g.dy + size_t(position[j + q]) * g.cols + size_t(u) * VEC);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if (j + q >= j1) continue;
#pragma unroll
            for (int c = 0; c < VEC; ++c) sum.v[c] += v[q].v[c];
            const unsigned key = keys[1 + j + q];
            const bool ends = keys[2 + j + q] != key;
            if (!ends && j + q + 1 < j1) continue;
            if (key < g.vocab) {
                if (ends && began) write_row<VEC>(g, key, u, sum);
                else store<VEC>(kept + (began ? g.pitch : 0), sum);
            }
            began = true;
#pragma unroll
            for (int c = 0; c < VEC; ++c) sum.v[c] = 0.f;
        }
    }
}

// Runs of more than one piece: what their first piece kept behind, and what every later one kept in front.
template <int VEC>
__global__ void __launch_bounds__(kGradThreads) embed_fold_kernel(Grad g) {
    const unsigned width = 1u << g.shift, groups = kGradThreads >> g.shift, lane = threadIdx.x & (width - 1);
    const unsigned piece = blockIdx.x / g.slabs * groups + (threadIdx.x >> g.shift), u = blockIdx.x % g.slabs * width + lane;
    if (piece + 1 >= g.pieces || u >= g.units) return;
    const unsigned begin = piece * kPiece, next = begin + kPiece, key = g.keys[next - 1];
    if (key >= g.vocab || g.keys[next] != key) return;
    if (begin && g.keys[begin - 1] == key && g.keys[begin] == key) return;  // began in front of this piece
    const unsigned end = next + lower_bound(g.keys + next, g.count - next, key + 1), last = (end - 1) / kPiece;
    const float *kept = g.kept + size_t(u) * VEC;
    Values<VEC> sum = load<VEC>(kept + (size_t(piece) * 2 + 1) * g.pitch);
    for (unsigned p = piece + 1; p <= last; p += 8) {
        Values<VEC> v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (p + q <= last) v[q] = load<VEC>(kept + size_t(p + q) * 2 * g.pitch);
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (p + q <= last)
#pragma unroll
                for (int c = 0; c < VEC; ++c) sum.v[c] += v[q].v[c];
    }
    write_row<VEC>(g, key, u, sum);
}

template <int VEC>
int32_t launch_grad(katsu_cuda_ctx *ctx, Grad g) {
    g.units = unsigned(g.cols / VEC);
    g.shift = 2;
    while ((1 << g.shift) < kGradThreads && (1u << g.shift) < g.units) ++g.shift;
    g.slabs = (g.units + (1u << g.shift) - 1) >> g.shift;
    const size_t groups = kGradThreads >> g.shift, piece_blocks = katsu_div_up(g.pieces, groups) * g.slabs;
    g.fill_rows = unsigned(std::min<size_t>(kGradThreads, std::max<size_t>(1, 16384 / g.cols)));
    const size_t fill_blocks = g.accumulate ? 0 : katsu_div_up(g.vocab, g.fill_rows);
    if (piece_blocks + fill_blocks > 0x7fffffffu)
        return katsu_set_error(KATSU_ERR_UNSUPPORTED, "%u tokens with rows of %zu values in one gradient", g.count, g.cols);
    g.piece_blocks = unsigned(piece_blocks);
    if (piece_blocks + fill_blocks)
        KATSU_LAUNCH(ctx, embed_grad_kernel<VEC>, unsigned(piece_blocks + fill_blocks), kGradThreads, 0, g);
    if (g.pieces > 1) KATSU_LAUNCH(ctx, embed_fold_kernel<VEC>, unsigned(piece_blocks), kGradThreads, 0, g);
    return KATSU_OK;
}

// Leaves the sorted keys and their positions in two of the four arrays of `count` words at `work`.
int32_t sort_tokens(katsu_cuda_ctx *ctx, const int *tokens, unsigned count, unsigned vocab, unsigned *work, const unsigned **keys,
                    const int **position) {
    unsigned *key_of_side[2] = {work, work + 2 * size_t(count)};
    int *position_of_side[2] = {reinterpret_cast<int *>(work + count), reinterpret_cast<int *>(work + 3 * size_t(count))};
    int side = 0;
    if (count <= kMostRanked) {
        KATSU_TRY(katsu_launch_chained(ctx, rank_kernel, (count + kRanked - 1) / kRanked, 256, 0, 1, tokens, count, vocab, key_of_side[0],
                                       position_of_side[0]));
    } else {
        unsigned *digits = work + 4 * size_t(count);
        const int bits = 32 - __builtin_clz(vocab), passes = (bits + 9) / 10, of_pass = (bits + passes - 1) / passes;
        const unsigned blocks = std::min<unsigned>(kSorters, (count + 2047) / 2048), tile = ((count + blocks - 1) / blocks + 255) / 256 * 256;
        const unsigned grid = (count + tile - 1) / tile;
        for (int pass = 0; pass < passes; ++pass, side ^= 1) {
            Pass p = {pass ? nullptr : tokens, key_of_side[side ^ 1], position_of_side[side ^ 1], count, vocab, tile, pass * of_pass, of_pass};
            KATSU_TRY(katsu_launch_chained(ctx, digits_kernel, grid, 256, 0, 1, p, digits));
            KATSU_TRY(katsu_launch_chained(ctx, scatter_kernel, grid, 256, 0, 1, p, static_cast<const unsigned *>(digits), key_of_side[side],
                                           position_of_side[side]));
        }
        side ^= 1;
    }
    *keys = key_of_side[side];
    *position = position_of_side[side];
    return KATSU_OK;
}

int32_t check(const katsu_cuda_ctx *ctx, size_t count, size_t vocab, size_t cols) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_REQUIRE(count <= 0x7fffffffu && vocab <= 0x7fffffffu && cols <= 0x3fffffffu, "tokens and vocab are below 2^31, cols below 2^30");
    KATSU_REQUIRE(vocab == 0 || cols <= SIZE_MAX / 8 / vocab, "the table is larger than addresses go");
    KATSU_REQUIRE(count == 0 || cols <= SIZE_MAX / 8 / count, "the rows are larger than addresses go");
    return KATSU_OK;
}

}  // namespace

extern "C" int32_t katsu_cuda_embed_fwd(katsu_cuda_ctx *ctx, const float *table, const int32_t *tokens, float scale, float *y,
                                        size_t count, size_t vocab, size_t cols) {
    KATSU_TRY(check(ctx, count, vocab, cols));
    if (count == 0 || cols == 0) return katsu_bind(ctx);
    KATSU_REQUIRE(tokens != nullptr && y != nullptr && (table != nullptr || vocab == 0), "null buffer");
    KATSU_REQUIRE(katsu_whole(table) && katsu_whole(tokens) && katsu_whole(y), "an address is not that of a whole element");
    KATSU_REQUIRE(!katsu_overlap(y, 4 * count * cols, table, 4 * vocab * cols) && !katsu_overlap(y, 4 * count * cols, tokens, 4 * count),
                  "y overlaps an input");
    KATSU_TRY(katsu_bind(ctx));
    return vectors(table, cols) && vectors(y, cols)
               ? launch_lookup<4, false>(ctx, table, nullptr, tokens, scale, y, count, vocab, 0, cols)
               : launch_lookup<1, false>(ctx, table, nullptr, tokens, scale, y, count, vocab, 0, cols);
}

extern "C" int32_t katsu_cuda_int8_embed(katsu_cuda_ctx *ctx, const int8_t *q, const float *rows_scale, const int32_t *tokens,
                                         float scale, float *y, size_t count, size_t vocab, size_t cols) {
    KATSU_TRY(check(ctx, count, vocab, cols));
    if (count == 0 || cols == 0) return katsu_bind(ctx);
    size_t pitch = 0;
    KATSU_TRY(katsu_cuda_int8_row_bytes(cols, &pitch));
    KATSU_REQUIRE(tokens != nullptr && y != nullptr && ((q != nullptr && rows_scale != nullptr) || vocab == 0), "null buffer");
    KATSU_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0, "an 8-bit matrix starts at a 16-byte aligned address");
    KATSU_REQUIRE(katsu_whole(rows_scale) && katsu_whole(tokens) && katsu_whole(y), "an address is not that of a whole element");
    const size_t bytes = 4 * count * cols;
    KATSU_REQUIRE(!katsu_overlap(y, bytes, q, vocab * pitch) && !katsu_overlap(y, bytes, rows_scale, 4 * vocab) &&
                      !katsu_overlap(y, bytes, tokens, 4 * count), "y overlaps an input");
    KATSU_TRY(katsu_bind(ctx));
    return vectors(y, cols) ? launch_lookup<4, true>(ctx, q, rows_scale, tokens, scale, y, count, vocab, pitch, cols)
                            : launch_lookup<1, true>(ctx, q, rows_scale, tokens, scale, y, count, vocab, pitch, cols);
}

extern "C" int32_t katsu_cuda_embed_bwd(katsu_cuda_ctx *ctx, const int32_t *tokens, const float *dy, float scale, float *dtable,
                                        size_t count, size_t vocab, size_t cols, int32_t accumulate) {
    KATSU_TRY(check(ctx, count, vocab, cols));
    if (vocab == 0 || cols == 0) return katsu_bind(ctx);
    KATSU_REQUIRE(dtable != nullptr && ((tokens != nullptr && dy != nullptr) || count == 0), "null buffer");
    KATSU_REQUIRE(katsu_whole(tokens) && katsu_whole(dy) && katsu_whole(dtable), "an address is not that of a whole element");
    KATSU_REQUIRE(!katsu_overlap(dtable, 4 * vocab * cols, dy, 4 * count * cols) && !katsu_overlap(dtable, 4 * vocab * cols, tokens, 4 * count),
                  "dtable overlaps an input");
    KATSU_TRY(katsu_bind(ctx));
    if (count == 0) return accumulate ? KATSU_OK : katsu_cuda_zero(ctx, dtable, vocab * cols);
    Grad g = {};
    g.dy = dy;
    g.dtable = dtable;
    g.scale = scale;
    g.count = unsigned(count);
    g.vocab = unsigned(vocab);
    g.pieces = unsigned(katsu_div_up(count, kPiece));
    g.accumulate = accumulate != 0;
    g.cols = cols;
    g.pitch = (cols + 3) / 4 * 4;
    const size_t sorting = (4 * count + size_t(kSorters) * kDigits + 3) / 4 * 4;
    float *work = nullptr;
    KATSU_TRY(katsu_scratch(ctx, sorting + size_t(g.pieces) * 2 * g.pitch, &work));
    g.kept = work + sorting;
    KATSU_TRY(sort_tokens(ctx, tokens, g.count, g.vocab, reinterpret_cast<unsigned *>(work), &g.keys, &g.position));
    return vectors(dy, cols) && vectors(dtable, cols) ? launch_grad<4>(ctx, g) : launch_grad<1>(ctx, g);
}
