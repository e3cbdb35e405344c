// Rows of a table for a list of tokens, and the gradient of the table.
//
//   y[i] = scale * table[t_i]                        dtable[v] (+)= scale * sum over i with t_i = v of dy[i]
//
// The lookup reads the rows of the tokens and writes y: HBM (8192 x 4096: 33 us, 5.8 TB/s).
//
// The gradient sorts the tokens (positions of one token in ascending order behind each other), cuts the sorted list into pieces of 8
// to 64 and adds up each piece on its own, whatever the tokens are: a token of a tenth of all positions costs what a thousand rare
// ones cost.  Runs that lie in one piece are written as they end; what a piece has of a run that began in front of it or goes on behind
// it is kept beside the table and folded in the pieces' order by a launch behind, in two steps where runs may be long.  Rows without
// a token get zeros from blocks of the pieces' launch.  No floating-point atomics: the same tokens give the same bits.  Bound: HBM for
// large gradients (65536 x 2048 into a table of as many rows: 154 us of 196, 7.0 TB/s with what L2 keeps; sorting 21, folding 19),
// three launches one behind the other for small ones (3001 x 515: 15.3 us).
#include <algorithm>

#include "common.cuh"
#include "launch.cuh"

namespace {

constexpr int kThreads = 256, kLookups = 8;  // of a lookup, and its blocks of an SM

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
// A row is `units` accesses of VEC values; 1 << shift threads share a row, four accesses each (a block's slab of 1024 accesses of
// it, where it is longer): a thread's four are on their way together (100 000 rows of 64 values: 10.5 us with one access a thread).
struct Rows {
    unsigned count, units, slabs;
    int shift;
};

Rows rows_of(size_t count, size_t units) {
    Rows r;
    r.count = unsigned(count);
    r.units = unsigned(units);
    r.shift = 0;
    while (r.shift < 8 && (size_t(4) << r.shift) < units) ++r.shift;
    r.slabs = unsigned(katsu_div_up(units, size_t(4) << r.shift));
    return r;
}

// INT8: the table's rows are int8_t of `pitch` bytes with a scale each, four values a load.
template <int VEC, bool INT8>
__global__ void __launch_bounds__(kThreads, kLookups) embed_kernel(const void *table, const float *rows_scale, const int *tokens, float scale,
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
            v[q] = load<VEC>(static_cast<const float *>(table) + size_t(token) * pitch + size_t(u) * VEC);
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

// Rows that are not whole 16-byte units: y is written by 16 bytes from its own boundary on, whatever rows these are of, and the
// table is read value by value.  Fewer than 2^32 values in all.
template <bool INT8>
__global__ void __launch_bounds__(kThreads, kLookups) embed_flat_kernel(const void *table, const float *rows_scale, const int *tokens, float scale,
                                                                        float *y, unsigned values, unsigned vocab, size_t pitch, unsigned cols, int waves) {
    if (!waves) launch_next();
    launch_wait();
    const unsigned lead = unsigned(reinterpret_cast<uintptr_t>(y) >> 2) & 3u;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        // places are counted from the boundary at or in front of y; those in front of it are numbers above `values`
        const unsigned long long place = 4ull * ((unsigned long long)blockIdx.x * (2 * kThreads) + q * kThreads + threadIdx.x);
        if (place >= (unsigned long long)values + lead) return;
        const unsigned first = unsigned(place) - lead;
        float v[4];
        unsigned row = (first < values ? first : 0) / cols, col = (first < values ? first : 0) - row * cols;
        if (first < values && cols - col >= 4) {  // four of one row
            const unsigned token = unsigned(tokens[row]);
            const size_t at = size_t(token) * pitch + col;
            const bool there = token < vocab;
            const float of_row = INT8 && there ? rows_scale[token] : 1.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (!there) v[c] = 0.f;
                else if (INT8) v[c] = (float(static_cast<const int8_t *>(table)[at + c]) * of_row) * scale;
                else v[c] = static_cast<const float *>(table)[at + c] * scale;
            }
            *reinterpret_cast<float4 *>(y + first) = make_float4(v[0], v[1], v[2], v[3]);
            continue;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            v[c] = 0.f;
            if (first + c >= values) continue;
            const unsigned token = unsigned(tokens[row]);
            if (token < vocab) {
                if (INT8) v[c] = (float(static_cast<const int8_t *>(table)[size_t(token) * pitch + col]) * rows_scale[token]) * scale;
                else v[c] = static_cast<const float *>(table)[size_t(token) * pitch + col] * scale;
            }
            if (++col == cols) {
                col = 0;
                ++row;
            }
        }
        if (first < values && values - first >= 4) {
            *reinterpret_cast<float4 *>(y + first) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (first + c < values) y[first + c] = v[c];
        }
    }
}

bool vectors(const void *p, size_t cols) { return cols % 4 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// pitch: bytes (8-bit rows) or values (others) from one row of the table to the next
template <bool INT8>
int32_t lookup(katsu_cuda_ctx *ctx, const void *table, const float *rows_scale, const int *tokens, float scale, float *y, size_t count,
               size_t vocab, size_t pitch, size_t cols) {
    const bool whole = vectors(y, cols) && (INT8 || vectors(table, cols));
    if (!whole && count * cols < 0xfffffff0u) {
        const size_t blocks = katsu_div_up(count * cols + 3, size_t(8) * kThreads);
        const bool waves = blocks > size_t(kLookups) * ctx->num_sms;
        return katsu_launch(ctx, !waves, embed_flat_kernel<INT8>, unsigned(blocks), kThreads, 0, 1, table, rows_scale, tokens, scale, y,
                            unsigned(count * cols), unsigned(vocab), pitch, unsigned(cols), int(waves));
    }
    const Rows rows = rows_of(count, whole ? cols / 4 : cols);
    const size_t blocks = katsu_div_up(count, kThreads >> rows.shift) * rows.slabs;
    if (blocks > 0x7fffffffu) return katsu_set_error(KATSU_ERR_UNSUPPORTED, "%zu rows of %zu values in one lookup", count, cols);
    const bool waves = blocks > size_t(kLookups) * ctx->num_sms;
    return katsu_launch(ctx, !waves, whole ? embed_kernel<4, INT8> : embed_kernel<1, INT8>, unsigned(blocks), kThreads, 0, 1, table, rows_scale,
                        tokens, scale, y, rows, unsigned(vocab), pitch, cols, int(waves));
}

// ---- sorting the tokens --------------------------------------------------------------------------------------------------
// keys[p] and position[p]: the tokens in ascending order, equal ones by position, what is no token (key `vocab`) last.
constexpr int kRanked = 32, kMostRanked = 8192;

__device__ __forceinline__ unsigned key_of(int token, unsigned vocab) { return min(unsigned(token), vocab); }

// Up to 8192 tokens: the place of a token is the number of tokens that belong in front of it.  A block counts for 32 of them,
// its warps over a sixteenth of the list each, 32 comparisons a lane for eight loads of 16 bytes that all lanes share: one launch
// (3001 tokens 6 us, 8192 13; two lists side by side in a warp, for twice the blocks, took twice the time).
constexpr int kRankThreads = 512, kRankBlocks = 2;  // blocks of an SM: all 256 of a list are resident, so that each launch may start early

__global__ void __launch_bounds__(kRankThreads, kRankBlocks) rank_kernel(const int *tokens, unsigned count, unsigned vocab, unsigned *keys, int *position) {
    __shared__ __align__(16) unsigned all[kMostRanked];
    __shared__ int partial[kRankThreads / 32][kRanked];
    launch_next();
    launch_wait();
    const unsigned tiles = (count + 31) / 32, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 4
    for (unsigned j = threadIdx.x; j < tiles * 32; j += kRankThreads) all[j] = j < count ? key_of(tokens[j], vocab) : 0xffffffffu;
    __syncthreads();
    const unsigned i = blockIdx.x * kRanked + lane, key = all[i];
    int before = 0;
    for (unsigned tile = warp; tile < tiles; tile += kRankThreads / 32) {
        const uint4 *of_tile = reinterpret_cast<const uint4 *>(all + 32 * tile);
        const unsigned limit = key + (tile < blockIdx.x ? 1 : 0);  // in front: equal ones count too
#pragma unroll
        for (unsigned q = 0; q < 8; ++q) {
            const uint4 k = of_tile[q];
            before += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
        }
        if (tile == blockIdx.x)
#pragma unroll
            for (unsigned q = 0; q < 8; ++q) {
                const uint4 k = of_tile[q];
                before += (k.x == key && 4 * q < lane) + (k.y == key && 4 * q + 1 < lane) + (k.z == key && 4 * q + 2 < lane) +
                          (k.w == key && 4 * q + 3 < lane);
            }
    }
    partial[warp][lane] = before;
    __syncthreads();
    if (warp != 0 || i >= count) return;
    int place = 0;
#pragma unroll
    for (int w = 0; w < kRankThreads / 32; ++w) place += partial[w][lane];
    keys[place] = key;
    position[place] = int(i);
}

// More: passes over digits of two to ten bits from the lowest on, a launch each, behind one that counts the first pass's digits; a
// pass counts those of the next where it puts the keys.  A block has `tile` of the keys, a multiple of kTile.
constexpr int kDigits = 1024, kSorters = 128, kTile = 2048;

struct Pass {
    const int *tokens;                              // first pass
    const unsigned *keys;                           // later ones
    const int *position;
    unsigned count, vocab, tile;
    int shift, bits;
};

__device__ __forceinline__ unsigned pass_key(const Pass &p, unsigned i) { return p.tokens ? key_of(p.tokens[i], p.vocab) : p.keys[i]; }

// digits[block][digit]: how many of the block's keys have the digit.  next: zeros, for the pass behind.
__global__ void __launch_bounds__(256, 1) digits_kernel(Pass p, unsigned *digits, unsigned *next) {
    __shared__ unsigned mine[kDigits];
    launch_next();
    const unsigned values = 1u << p.bits, mask = values - 1;
    for (unsigned d = threadIdx.x; d < values; d += 256) mine[d] = 0;
    __syncthreads();
    launch_wait();
    const unsigned begin = blockIdx.x * p.tile, end = min(p.count, begin + p.tile);
#pragma unroll 8
    for (unsigned i = begin + threadIdx.x; i < end; i += 256) atomicAdd(&mine[(pass_key(p, i) >> p.shift) & mask], 1u);
    __syncthreads();
    for (unsigned d = threadIdx.x; d < values; d += 256) {
        digits[blockIdx.x * values + d] = mine[d];
        next[blockIdx.x * values + d] = 0;
    }
}

// Moves the block's keys to their places, and counts the next pass's digits there (next, null: this is the last one; behind: zeros
// for the one behind that).  A warp takes an eighth of them in order, so that equal digits keep theirs; eight keys a lane are on their
// way together.  65536 tokens: 8 to 10 us a pass, most of it the chain of loads, counts and scans; counting 3.
__global__ void __launch_bounds__(256, 1) scatter_kernel(Pass p, const unsigned *digits, unsigned *next, unsigned *behind, unsigned *keys, int *position) {
    __shared__ __align__(16) unsigned place[8][kDigits];
    __shared__ __align__(16) unsigned all[kDigits], front[kDigits];
    __shared__ unsigned sums[8];
    launch_next();
    const unsigned values = 1u << p.bits, mask = values - 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (unsigned d = lane; d < values; d += 32) place[warp][d] = 0;
    for (unsigned d = threadIdx.x; d < kDigits; d += 256) all[d] = front[d] = 0;
    __syncthreads();
    launch_wait();
    const unsigned share = p.tile / 8, begin = min(p.count, blockIdx.x * p.tile + warp * share), end = min(p.count, begin + share);
    if (behind)
        for (unsigned d = threadIdx.x; d < values; d += 256) behind[blockIdx.x * values + d] = 0;
    unsigned key[8];
    int at[8];
    auto fetch = [&](unsigned from) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const unsigned i = from + 32 * q + lane;
            key[q] = i < end ? pass_key(p, i) : 0xffffffffu;  // (no key: keys are at most 2^31 - 1)
            at[q] = p.tokens ? int(i) : i < end ? p.position[i] : 0;
        }
    };
    fetch(begin);
    // keys of each digit in all blocks and in those in front of this one: four digits a thread, the blocks shared out among threads
    const unsigned quads = values / 4, parts = 256 / quads, quad = threadIdx.x % quads;
    uint4 sum_all = make_uint4(0, 0, 0, 0), sum_front = sum_all;
    for (unsigned b0 = threadIdx.x / quads; b0 < gridDim.x; b0 += 8 * parts) {
        uint4 n[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const unsigned b = b0 + q * parts;
            n[q] = b < gridDim.x ? *reinterpret_cast<const uint4 *>(digits + size_t(b) * values + 4 * quad) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            sum_all.x += n[q].x, sum_all.y += n[q].y, sum_all.z += n[q].z, sum_all.w += n[q].w;
            if (b0 + q * parts < blockIdx.x) sum_front.x += n[q].x, sum_front.y += n[q].y, sum_front.z += n[q].z, sum_front.w += n[q].w;
        }
    }
    const unsigned of_all[4] = {sum_all.x, sum_all.y, sum_all.z, sum_all.w}, of_front[4] = {sum_front.x, sum_front.y, sum_front.z, sum_front.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        atomicAdd(&all[4 * quad + q], of_all[q]);
        atomicAdd(&front[4 * quad + q], of_front[q]);
    }
    for (unsigned from = begin; from < end; from += 256) {
        if (from != begin) fetch(from);
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (key[q] != 0xffffffffu) atomicAdd(&place[warp][(key[q] >> p.shift) & mask], 1u);
    }
    __syncthreads();
    const uint4 mine = reinterpret_cast<const uint4 *>(all)[threadIdx.x];  // zeros behind the digits
    unsigned scan = mine.x + mine.y + mine.z + mine.w;
    const unsigned sum = scan;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned other = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= unsigned(o)) scan += other;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    unsigned first = scan - sum;
    for (unsigned w = 0; w < warp; ++w) first += sums[w];
    if (4 * threadIdx.x < values) {
        const uint4 in_front = reinterpret_cast<const uint4 *>(front)[threadIdx.x];
        uint4 from = make_uint4(first + in_front.x, first + mine.x + in_front.y, first + mine.x + mine.y + in_front.z,
                                first + mine.x + mine.y + mine.z + in_front.w);
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            uint4 *at = reinterpret_cast<uint4 *>(place[w]) + threadIdx.x;
            const uint4 n = *at;
            *at = from;
            from.x += n.x, from.y += n.y, from.z += n.z, from.w += n.w;
        }
    }
    __syncthreads();
    const bool again = end - begin > 256;
    for (unsigned from = begin; from < end; from += 256) {
        if (again) fetch(from);
        unsigned same[8];  // lanes with the same digit, by a vote on each of its bits: matching takes a step for each different one
#pragma unroll
        for (int q = 0; q < 8; ++q) same[q] = __ballot_sync(0xffffffffu, key[q] != 0xffffffffu);
        for (int bit = p.shift; bit < p.shift + p.bits; ++bit)
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const unsigned ones = __ballot_sync(0xffffffffu, key[q] >> bit & 1);
                same[q] &= key[q] >> bit & 1 ? ones : ~ones;
            }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const bool valid = key[q] != 0xffffffffu;
            const unsigned digit = (key[q] >> p.shift) & mask, ahead = __popc(same[q] & ((1u << lane) - 1));
            unsigned to = 0;
            if (valid) to = place[warp][digit] + ahead;
            __syncwarp();
            if (valid && ahead == 0) place[warp][digit] = to + __popc(same[q]);
            __syncwarp();
            if (!valid) continue;
            keys[to] = key[q];
            position[to] = at[q];
            if (next) atomicAdd(next + size_t(to / p.tile) * values + (key[q] >> (p.shift + p.bits) & mask), 1u);
        }
    }
}

// ---- the gradient ----------------------------------------------------------------------------------------------------------
constexpr int kGradThreads = 128, kMostPiece = 64, kDirect = 256;
// Blocks of an SM that the gradient's launches count with, where they ask whether one may start early; its kernels leave registers for
// these and more.
constexpr int kGradBlocks = 4, kPieceBlocks = 8, kAddBlocks = 5, kFoldBlocks = 5;
// (few tokens of odd rows: 9 to 12 within 5 % of each other, 16, which spills, 200 tokens x 101 added 7.5 us instead of 5.9)
constexpr int direct_blocks(bool whole, bool add) { return whole ? 8 : add ? 10 : 12; }
static_assert(std::min({kPieceBlocks, kAddBlocks, kFoldBlocks, direct_blocks(true, true)}) >= kGradBlocks,
              "launches that start early have all their blocks resident");
constexpr int kApart = 2;

struct Grad {
    const int *tokens;  // few tokens: unsorted
    const unsigned *keys;
    const int *position;
    const float *dy;
    float *dtable, *kept;  // kept [piece][2][pitch]: of the run that began in front; of the one that goes on behind
    float scale;
    unsigned count, vocab, units, slabs, piece, pieces, piece_blocks, fill_rows;
    int shift, fill_shift, waves;
    unsigned parts;  // of a run that are folded side by side
    bool accumulate, bundles;
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

// A thread's N values of a row, in slab `slab` of it and at place `lane` of the group: 16 bytes of rows that are whole 16-byte units
// (WHOLE), else kApart values a group's width apart, so that a warp's accesses lie side by side.  One, two and four of them: 91, 75 and
// 72 us for 30 000 rows of 1001, 58, 65 and 84 for 100 000 rows of 61 (longer pieces than today's, with which two take 65 us of 30 000).
template <bool WHOLE, int N>
struct Part {
    size_t at;
    unsigned step;
    int count;  // how many of the N there are

    __device__ __forceinline__ Part(const Grad &g, unsigned slab, unsigned lane) {
        step = 1u << g.shift;
        if (WHOLE) {
            const unsigned u = (slab << g.shift) + lane;
            at = 4 * size_t(u);
            count = u < g.units ? N : 0;
        } else {
            at = size_t(slab) * N * step + lane;
            count = at < g.cols ? int(min((unsigned(g.cols - at) + step - 1) >> g.shift, unsigned(N))) : 0;
        }
    }
    __device__ __forceinline__ Values<N> load(const float *row) const {
        if constexpr (WHOLE) return ::load<4>(row + at);
        Values<N> r;
#pragma unroll
        for (int c = 0; c < N; ++c) r.v[c] = c < count ? row[at + c * step] : 0.f;
        return r;
    }
    __device__ __forceinline__ void store(float *row, const Values<N> &r) const {
        if constexpr (WHOLE) ::store<4>(row + at, r);
        else
#pragma unroll
            for (int c = 0; c < N; ++c)
                if (c < count) row[at + c * step] = r.v[c];
    }
};

__device__ __forceinline__ float *row_of(const Grad &g, unsigned key) { return g.dtable + size_t(key) * g.cols; }

template <int N>
__device__ __forceinline__ Values<N> zero_values() {
    Values<N> r;
#pragma unroll
    for (int c = 0; c < N; ++c) r.v[c] = 0.f;
    return r;
}

template <int N>
__device__ __forceinline__ void add_values(Values<N> *sum, const Values<N> &v) {
#pragma unroll
    for (int c = 0; c < N; ++c) sum->v[c] += v.v[c];
}

// sum = scale * sum, added to what the table has where that is asked for
template <bool WHOLE, int N, bool ADD>
__device__ __forceinline__ void write_row(const Grad &g, const Part<WHOLE, N> &part, float *row, Values<N> sum, const Values<N> &old) {
#pragma unroll
    for (int c = 0; c < N; ++c) sum.v[c] = ADD ? fmaf(g.scale, sum.v[c], old.v[c]) : g.scale * sum.v[c];
    part.store(row, sum);
}

// Zeros for rows row0 .. row0 + rows - 1 but for those that are `there`, by 16 bytes from the first boundary of a row on.
__device__ __forceinline__ void fill_rows(const Grad &g, const bool *there, unsigned row0, unsigned rows) {
    const unsigned width = 1u << g.fill_shift, groups = kGradThreads >> g.fill_shift, lane = threadIdx.x & (width - 1);
    for (unsigned r = threadIdx.x >> g.fill_shift; r < rows; r += groups) {
        if (there[r]) continue;
        float *row = g.dtable + size_t(row0 + r) * g.cols;
        const unsigned cols = unsigned(g.cols), head = min(cols, (0u - unsigned(reinterpret_cast<uintptr_t>(row) >> 2)) & 3u), units = (cols - head) / 4;
        for (unsigned c = lane; c < head; c += width) row[c] = 0.f;
        float4 *body = reinterpret_cast<float4 *>(row + head);
        for (unsigned u = lane; u < units; u += width) body[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (unsigned c = head + 4 * units + lane; c < cols; c += width) row[c] = 0.f;
    }
}

// Up to kDirect tokens, without sorting: a group of 1 << shift threads takes the run of one token, if that is its first place.
template <bool WHOLE, int N, bool ADD>
__global__ void __launch_bounds__(kGradThreads, direct_blocks(WHOLE, ADD)) embed_direct_kernel(Grad g) {
    __shared__ __align__(16) unsigned keys[kDirect];
    __shared__ bool there[kGradThreads];
    if (!g.waves) launch_next();
    launch_wait();
    for (unsigned j = threadIdx.x; j < kDirect; j += kGradThreads) keys[j] = j < g.count ? key_of(g.tokens[j], g.vocab) : 0xffffffffu;
    there[threadIdx.x] = false;
    __syncthreads();
    if (blockIdx.x >= g.piece_blocks) {
        const unsigned row0 = (blockIdx.x - g.piece_blocks) * g.fill_rows, rows = min(g.fill_rows, g.vocab - row0);
        for (unsigned j = threadIdx.x; j < kDirect; j += kGradThreads)
            if (keys[j] - row0 < rows) there[keys[j] - row0] = true;
        __syncthreads();
        fill_rows(g, there, row0, rows);
        return;
    }
    const unsigned groups = kGradThreads >> g.shift, i = blockIdx.x / g.slabs * groups + (threadIdx.x >> g.shift);
    const Part<WHOLE, N> part(g, blockIdx.x % g.slabs, threadIdx.x & ((1u << g.shift) - 1));
    if (i >= g.count || part.count == 0) return;
    const unsigned key = keys[i];
    if (key >= g.vocab) return;
    // places of the token: the next one from `from` on in `same`, the 64 places of one word after the other
    auto word = [&](unsigned from) {
        unsigned long long same = 0;
#pragma unroll 4
        for (unsigned j = 0; j < 64; j += 4) {
            const uint4 k = *reinterpret_cast<const uint4 *>(keys + from + j);
            same |= (unsigned long long)((k.x == key) | (k.y == key) << 1 | (k.z == key) << 2 | (k.w == key) << 3) << j;
        }
        return same;
    };
    unsigned from = i & ~63u;
    unsigned long long same = word(from);
    if (same << (63 - (i & 63)) << 1) return;  // an earlier place, in this word or in those in front of it
    for (unsigned front = 0; front < from; front += 64)
        if (word(front)) return;
    float *dst = row_of(g, key);
    const Values<N> old = ADD ? part.load(dst) : zero_values<N>();
    Values<N> sum = zero_values<N>();
    for (;;) {
        while (!same && from + 64 < g.count) same = word(from += 64);
        if (!same) break;
        Values<N> v[8];
        int taken = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if (!same) continue;
            v[q] = part.load(g.dy + size_t(from + __ffsll((long long)same) - 1) * g.cols);
            same &= same - 1;
            taken = q + 1;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (q < taken)
                add_values(&sum, v[q]);
    }
    write_row<WHOLE, N, ADD>(g, part, dst, sum, old);
}

// Blocks 0 .. piece_blocks - 1: a group of 1 << shift threads adds up a piece (a slab of 1 << shift accesses of its rows); the
// blocks behind them write zeros to fill_rows rows of the table each, but for those of tokens that are there.
template <bool WHOLE, int N, bool ADD>
__global__ void __launch_bounds__(kGradThreads, ADD ? kAddBlocks : kPieceBlocks) embed_grad_kernel(Grad g) {
    const unsigned width = 1u << g.shift, groups = kGradThreads >> g.shift, mine = threadIdx.x >> g.shift, lane = threadIdx.x & (width - 1);
    extern __shared__ unsigned keys[];  // of the block's pieces, their positions behind them
    int *position = reinterpret_cast<int *>(keys + groups * g.piece + 2);
    __shared__ bool there[kGradThreads];
    if (!g.waves) launch_next();
    launch_wait();
    if (blockIdx.x >= g.piece_blocks) {
        const unsigned row0 = (blockIdx.x - g.piece_blocks) * g.fill_rows, rows = min(g.fill_rows, g.vocab - row0);
        if (threadIdx.x < rows) {
            const unsigned key = row0 + threadIdx.x, at = lower_bound(g.keys, g.count, key);
            there[threadIdx.x] = at < g.count && g.keys[at] == key;
        }
        __syncthreads();
        fill_rows(g, there, row0, rows);
        return;
    }
    const unsigned slab = blockIdx.x % g.slabs, piece0 = blockIdx.x / g.slabs * groups, begin0 = piece0 * g.piece;
    const unsigned staged = min(groups * g.piece, g.count - begin0);
    // keys[1 + j] is that of place begin0 + j; one in front and one behind as well, ~0 where there is none
    for (unsigned j = threadIdx.x; j < staged; j += kGradThreads) {
        keys[1 + j] = g.keys[begin0 + j];
        position[j] = g.position[begin0 + j];
    }
    if (threadIdx.x == 0) keys[0] = begin0 ? g.keys[begin0 - 1] : ~0u;
    if (threadIdx.x == 1) keys[1 + staged] = begin0 + staged < g.count ? g.keys[begin0 + staged] : ~0u;
    __syncthreads();
    const unsigned piece = piece0 + mine, j0 = mine * g.piece;
    const Part<WHOLE, N> part(g, slab, lane);
    if (piece >= g.pieces || part.count == 0) return;
    const unsigned j1 = min(staged, j0 + g.piece);
    float *kept = g.kept + size_t(piece) * 2 * g.pitch;
    bool began = keys[j0] != keys[j0 + 1];  // the current run began in this piece
    Values<N> sum = zero_values<N>();
    for (unsigned j = j0; j < j1; j += 8) {
        Values<N> v[8], old[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (j + q < j1) v[q] = part.load(g.dy + size_t(position[j + q]) * g.cols);
        if (ADD)  // rows that end here, asked for with the others: one by one they took a trip to memory each
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (j + q < j1 && keys[2 + j + q] != keys[1 + j + q] && keys[1 + j + q] < g.vocab)
                    old[q] = part.load(row_of(g, keys[1 + j + q]));
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            if (j + q >= j1) continue;
            add_values(&sum, v[q]);
            const unsigned key = keys[1 + j + q];
            const bool ends = keys[2 + j + q] != key;
            if (!ends && j + q + 1 < j1) continue;
            if (key < g.vocab) {
                if (ends && began) write_row<WHOLE, N, ADD>(g, part, row_of(g, key), sum, old[q]);
                else part.store(kept + (began ? g.pitch : 0), sum);
            }
            began = true;
            sum = zero_values<N>();
        }
    }
}

// Long runs (a padding token is half of a batch): kBundle pieces that one run fills, from a multiple of kBundle on, are added up into
// the place of the first one, by as many blocks as there are such bundles.  Where the run fills them, both kernels find the same.
constexpr unsigned kBundle = 32;

__device__ __forceinline__ bool bundle_of_run(const Grad &g, unsigned first, unsigned key) {
    const unsigned long long end = ((unsigned long long)first + kBundle) * g.piece;
    return end <= g.count && g.keys[end - 1] == key;  // (a piece of the run is `first`, and not its first one)
}

// The sum of what the pieces kept in front, sixteen on their way together.  next(&piece): whether there is another one, and which.
template <bool WHOLE, int N, typename Next>
__device__ __forceinline__ void add_kept(const Grad &g, const Part<WHOLE, N> &part, Values<N> *sum, Next &&next) {
    for (bool more = true; more;) {
        Values<N> v[16];
        int taken = 0;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            unsigned piece;
            more = more && next(&piece);
            if (!more) continue;
            v[q] = part.load(g.kept + size_t(piece) * 2 * g.pitch);
            taken = q + 1;
        }
#pragma unroll
        for (int q = 0; q < 16; ++q)
            if (q < taken)
                add_values(sum, v[q]);
    }
}

template <bool WHOLE, int N>
__global__ void __launch_bounds__(kGradThreads, kFoldBlocks) embed_bundle_kernel(Grad g) {
    const unsigned groups = kGradThreads >> g.shift;
    if (!g.waves) launch_next();
    launch_wait();
    const unsigned first = (blockIdx.x / g.slabs * groups + (threadIdx.x >> g.shift)) * kBundle;
    const Part<WHOLE, N> part(g, blockIdx.x % g.slabs, threadIdx.x & ((1u << g.shift) - 1));
    if (first == 0 || first >= g.pieces || part.count == 0) return;
    const unsigned key = g.keys[first * g.piece];
    if (key >= g.vocab || g.keys[first * g.piece - 1] != key || !bundle_of_run(g, first, key)) return;
    Values<N> sum = zero_values<N>();
    unsigned at = first;
    add_kept(g, part, &sum, [&](unsigned *piece) {
        *piece = at++;
        return *piece < first + kBundle;
    });
    part.store(g.kept + size_t(first) * 2 * g.pitch, sum);
}

// Threads of a group, and slabs of a row, at n values a thread.
struct Width {
    unsigned units, slabs;
    int shift;
};

constexpr Width width_of(size_t cols, size_t n) {
    Width w = {unsigned((cols + n - 1) / n), 1, 2};
    while ((1 << w.shift) < kGradThreads && (1u << w.shift) < w.units) ++w.shift;
    w.slabs = (w.units + (1u << w.shift) - 1) >> w.shift;
    return w;
}

// Parts of a run that its fold's warp adds up side by side: as many as rows of either kind have groups in a warp (the order is that of
// sizes).  A lane takes part fold_part(lane, shift), and none where that is not below the parts: rows that are whole 16-byte units have
// groups of half the size.
constexpr unsigned fold_parts(size_t cols) { return 32u >> std::min(5, width_of(cols, kApart).shift); }
__host__ __device__ constexpr unsigned fold_part(unsigned lane, int shift) { return lane >> shift; }

// Every value of a part of a run has one lane, whatever rows of up to a warp's width are, and there is a lane for all of them.
constexpr bool folds_each_value_once(size_t cols, size_t n) {
    const Width width = width_of(cols, n);
    for (unsigned part = 0; part < fold_parts(cols); ++part)
        for (unsigned unit = 0; unit < width.units; ++unit) {
            int lanes = 0;
            for (unsigned lane = 0; lane < 32; ++lane)
                lanes += fold_part(lane, width.shift) == part && (lane & ((1u << width.shift) - 1)) == unit;
            if (lanes != 1) return false;
        }
    return true;
}

constexpr bool folds_of_a_warp_are_right() {
    for (size_t cols = 1; cols <= 32 * kApart; ++cols)
        if (!folds_each_value_once(cols, kApart) || (cols % 4 == 0 && !folds_each_value_once(cols, 4))) return false;
    return true;
}
static_assert(folds_of_a_warp_are_right(), "a value of a run is folded by one lane");

// Runs of more than one piece: what their first piece kept behind, and what every later one (or bundle) kept in front.  A run has a
// group of threads, a warp at least: of rows of fewer threads as many neighbouring parts of the run as fit there are added up at once
// (100 000 x 16: 8 us; 32 where a run had four threads that looked at four pieces at a time).
template <bool WHOLE, int N, bool ADD>
__global__ void __launch_bounds__(kGradThreads, kFoldBlocks) embed_fold_kernel(Grad g) {
    const int shift = max(g.shift, 5);
    const unsigned groups = kGradThreads >> shift, lane = threadIdx.x & 31, width = 1u << g.shift;
    if (!g.waves) launch_next();
    launch_wait();
    const unsigned piece = blockIdx.x / g.slabs * groups + (threadIdx.x >> shift);
    const unsigned begin = piece * g.piece, next = begin + g.piece;
    if (piece + 1 >= g.pieces) return;
    const unsigned front = begin ? g.keys[begin - 1] : ~0u, first = g.keys[begin], key = g.keys[next - 1], behind = g.keys[next];
    if (key != behind || key >= g.vocab || (front == key && first == key)) return;  // (all threads of the group) not a run that began here and goes on
    // the last piece that begins with the token: 32 pieces at a time, from one step to the next 32 times as far, and back
    unsigned last = piece + 1, step = 1;
    auto through = [&] {
        const unsigned long long p = last + (lane + 1ull) * step;
        return unsigned(__popc(__ballot_sync(~0u, p < g.pieces && g.keys[p * g.piece] == key)));
    };
    unsigned far = through();
    for (;;) {
        last += far * step;
        if (far < 32) break;
        step *= 32;
        far = through();
    }
    while (step > 1) {
        step /= 32;
        last += through() * step;
    }
    const Part<WHOLE, N> part(g, blockIdx.x % g.slabs, threadIdx.x & (width - 1));
    const unsigned parts = g.parts, mine = fold_part(lane, g.shift);
    const bool there = part.count != 0 && mine < parts;
    const unsigned base = g.bundles ? (piece + 1) / kBundle * kBundle : piece + 1, bundle = g.bundles ? kBundle : 1;
    const unsigned share = ((last - base) / parts / bundle + 1) * bundle;
    float *dst = row_of(g, key);
    const Values<N> old = ADD && there && mine == 0 ? part.load(dst) : zero_values<N>();
    Values<N> sum = there && mine == 0 ? part.load(g.kept + (size_t(piece) * 2 + 1) * g.pitch) : zero_values<N>();
    unsigned at = max(piece + 1, base + mine * share);
    const unsigned end = min(last, base + mine * share + share - 1);
    if (there)
        add_kept(g, part, &sum, [&](unsigned *p) {
            *p = at;
            const bool bundled = g.bundles && at % kBundle == 0 && (at + kBundle <= last || (at + kBundle - 1 == last && bundle_of_run(g, at, key)));
            at += bundled ? kBundle : 1;
            return *p <= end;
        });
    if (parts > 1)
        for (unsigned o = parts * width / 2; o >= width; o >>= 1) {
            Values<N> other;
#pragma unroll
            for (int c = 0; c < N; ++c) other.v[c] = __shfl_xor_sync(~0u, sum.v[c], o);
            add_values(&sum, other);
        }
    if (there && mine == 0) write_row<WHOLE, N, ADD>(g, part, dst, sum, old);
}

template <bool WHOLE, int N, bool ADD>
int32_t launch_grad(katsu_cuda_ctx *ctx, Grad g) {
    const Width width = width_of(g.cols, N);
    g.units = width.units;
    g.shift = width.shift;
    g.slabs = width.slabs;
    const size_t groups = kGradThreads >> g.shift, piece_blocks = katsu_div_up(g.pieces, groups) * g.slabs;
    // zeros: about 64 KiB a block, less where that leaves SMs without one; two accesses of a thread to a row
    const size_t shared_out = katsu_div_up(g.vocab, size_t(8) * ctx->num_sms);
    g.fill_rows = unsigned(std::max<size_t>(1, std::min({size_t(kGradThreads), 16384 / g.cols, shared_out})));
    g.fill_shift = 0;
    while ((1 << g.fill_shift) < kGradThreads && (size_t(8) << g.fill_shift) < g.cols) ++g.fill_shift;
    const size_t fill_blocks = ADD ? 0 : katsu_div_up(g.vocab, g.fill_rows), blocks = piece_blocks + fill_blocks;
    if (blocks > 0x7fffffffu)
        return katsu_set_error(KATSU_ERR_UNSUPPORTED, "%u tokens with rows of %zu values in one gradient", g.count, g.cols);
    g.piece_blocks = unsigned(piece_blocks);
    const size_t resident = size_t(kGradBlocks) * ctx->num_sms;
    g.waves = blocks > resident;
    if (g.tokens) return katsu_launch(ctx, !g.waves, embed_direct_kernel<WHOLE, N, ADD>, unsigned(blocks), kGradThreads, 0, 1, g);
    KATSU_TRY(katsu_launch(ctx, !g.waves, embed_grad_kernel<WHOLE, N, ADD>, unsigned(blocks), kGradThreads, (2 * groups * g.piece + 2) * sizeof(unsigned), 1, g));
    if (g.pieces == 1) return KATSU_OK;
    // Bundles are another launch, for which lists without a very frequent token pay 1 to 1.5 us (16384 x 512: 32.8 to 34.0) unless they are
    // long (100 000 x 64: 48 to 39).  Where one token is 70 % of the list they take 16384 x 512 from 58 to 35 us, 100 000 x 64 from 214 to
    // 42; below 512 pieces for each part of a run still 8192 x 512 from 41 to 34, but the fold is short enough to do without.
    const int fold_shift = std::max(g.shift, 5);
    g.parts = fold_parts(g.cols);
    g.bundles = g.pieces >= 512 * g.parts;
    if (g.bundles) {
        const size_t bundle_blocks = katsu_div_up(katsu_div_up(g.pieces, kBundle), groups) * g.slabs;
        g.waves = bundle_blocks > resident;
        KATSU_TRY(katsu_launch(ctx, !g.waves, embed_bundle_kernel<WHOLE, N>, unsigned(bundle_blocks), kGradThreads, 0, 1, g));
    }
    const size_t fold_blocks = katsu_div_up(g.pieces, size_t(kGradThreads) >> fold_shift) * g.slabs;
    if (fold_blocks > 0x7fffffffu)
        return katsu_set_error(KATSU_ERR_UNSUPPORTED, "%u tokens with rows of %zu values in one gradient", g.count, g.cols);
    g.waves = fold_blocks > resident;
    return katsu_launch(ctx, !g.waves, embed_fold_kernel<WHOLE, N, ADD>, unsigned(fold_blocks), kGradThreads, 0, 1, g);
}

int32_t launch_grad_for(katsu_cuda_ctx *ctx, const Grad &g, bool whole) {
    if (g.accumulate) return whole ? launch_grad<true, 4, true>(ctx, g) : launch_grad<false, kApart, true>(ctx, g);
    return whole ? launch_grad<true, 4, false>(ctx, g) : launch_grad<false, kApart, false>(ctx, g);
}

// Leaves the sorted keys and their positions in two of the four arrays of `count` words at `work`.
int32_t sort_tokens(katsu_cuda_ctx *ctx, const int *tokens, unsigned count, unsigned vocab, unsigned *work, const unsigned **keys,
                    const int **position) {
    unsigned *key_of_side[2] = {work, work + 2 * size_t(count)};
    int *position_of_side[2] = {reinterpret_cast<int *>(work + count), reinterpret_cast<int *>(work + 3 * size_t(count))};
    int side = 0;
    if (count <= kMostRanked) {
        KATSU_TRY(katsu_launch_chained(ctx, rank_kernel, (count + kRanked - 1) / kRanked, kRankThreads, 0, 1, tokens, count, vocab, key_of_side[0],
                                       position_of_side[0]));
    } else {
        unsigned *digits = work + 4 * size_t(count);
        const int bits = 32 - __builtin_clz(vocab), passes = (bits + 9) / 10, of_pass = std::max(2, (bits + passes - 1) / passes);
        const unsigned blocks = std::min<unsigned>(kSorters, (count + kTile - 1) / kTile), tile = ((count + blocks - 1) / blocks + kTile - 1) / kTile * kTile;
        const unsigned grid = (count + tile - 1) / tile;
        unsigned *of_pass_digits[3] = {digits, digits + kSorters * kDigits, digits + 2 * kSorters * kDigits};
        for (int pass = 0; pass < passes; ++pass, side ^= 1) {
            Pass p = {pass ? nullptr : tokens, key_of_side[side ^ 1], position_of_side[side ^ 1], count, vocab, tile, pass * of_pass, of_pass};
            if (pass == 0) KATSU_TRY(katsu_launch_chained(ctx, digits_kernel, grid, 256, 0, 1, p, of_pass_digits[0], of_pass_digits[1]));
            KATSU_TRY(katsu_launch_chained(ctx, scatter_kernel, grid, 256, 0, 1, p, static_cast<const unsigned *>(of_pass_digits[pass % 3]),
                                           pass + 1 < passes ? of_pass_digits[(pass + 1) % 3] : nullptr,
                                           pass + 2 < passes ? of_pass_digits[(pass + 2) % 3] : nullptr, key_of_side[side], position_of_side[side]));
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
    return lookup<false>(ctx, table, nullptr, tokens, scale, y, count, vocab, cols, cols);
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
    return lookup<true>(ctx, q, rows_scale, tokens, scale, y, count, vocab, pitch, cols);
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
    g.accumulate = accumulate != 0;
    g.cols = cols;
    g.pitch = (cols + 3) / 4 * 4;
    const bool whole = vectors(dy, cols) && vectors(dtable, cols);
    if (count <= kDirect) {
        g.tokens = tokens;
        g.pieces = g.count;
        return launch_grad_for(ctx, g, whole);
    }
    // A piece is a chain of loads, eight at a time: short ones, as long as their blocks are not more than three rounds.  Where the rows
    // are many bytes, pieces below 32 write too many sums beside the table.  (Sizes decide, not addresses: the order of the sums is theirs.)
    const Width width = width_of(cols, cols % 4 ? kApart : 4);
    g.piece = count * cols >= size_t(1) << 22 ? 32 : count <= 4096 ? 8 : 16;
    while (g.piece < kMostPiece && katsu_div_up(katsu_div_up(count, g.piece), kGradThreads >> width.shift) * width.slabs > size_t(16) * ctx->num_sms)
        g.piece *= 2;
    g.pieces = unsigned(katsu_div_up(count, g.piece));
    const size_t sorting = 4 * count + 3 * size_t(kSorters) * kDigits;
    float *work = nullptr;
    KATSU_TRY(katsu_scratch(ctx, sorting + size_t(g.pieces) * 2 * g.pitch, &work));
    g.kept = work + sorting;
    KATSU_TRY(sort_tokens(ctx, tokens, g.count, g.vocab, reinterpret_cast<unsigned *>(work), &g.keys, &g.position));
    return launch_grad_for(ctx, g, whole);
}
