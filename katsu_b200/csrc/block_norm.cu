// The norms in front of and behind a block, with the block's gate and the residual scale: forward and backward.
//
//   u = N(h; post) or h        r = x + scale * gate * u        n = N(r; pre)
//   N(v; w, b) = (v - m) * rstd * w + b,  rstd = 1 / sqrt(mean((v - m)^2) + eps),  m = mean(v) (layer) or 0 (RMS)
//
// With v^ = (v - m) * rstd and a gradient g of N(v; w, b), a = g w:
//
//   dw = sum over rows of g v^,   db = sum of g,   dv = rstd * (a - v^ mean(a v^) - mean(a))     (RMS: no last term)
//
// so a row of the backward takes mean(a (v - m)) and mean(a) beside the statistics themselves, one round of sums for both:
//
//   D  = dr + dv of N(r; pre) under dn                        = dx
//   du = scale * gate * D,   dgate = sum of scale * D * u,    dh = dv of N(h; post) under du
//
// A row belongs to one warp or block, in the backward above 4096 values to a cluster of blocks.  Sums over rows (weights, biases,
// gate) are kept a block and folded by a second launch in a fixed order.  Variances are of differences from the mean, in a round of their own: mean(v^2) - m^2 in 32 bits would lose a
// row whose mean is a thousand times its spread.
#include <math.h>

#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "launch.cuh"
#include "sm100.cuh"
#include "sm100_pair.cuh"

using namespace sm100;

namespace {

struct Forward {
    const float *x, *h, *gate, *post_w, *post_b, *pre_w, *pre_b;
    float *r, *n;
    float scale, eps;
    unsigned long long rows, rows_per_gate;
    int cols, ahead;
};

// Sums over rows, in the order of the partial results.
enum Sum { DPRE_W, DPRE_B, DPOST_W, DPOST_B, DGATE, SUMS };

struct Backward {
    const float *r, *h, *gate, *post_w, *post_b, *pre_w, *dr, *dn;
    float *dx, *dh;
    float *dgate;         // where a row's own gate is, or whole groups are one block's; else among the partial results
    float *partial[SUMS];  // [blocks][cols], null: not asked for
    float scale, eps;
    unsigned long long rows, rows_per_gate;
    int cols;
    // Rows go to blocks in groups of equal length: `groups` of them, cut into `slices` blocks each, or several to a block.
    unsigned long long groups;
    int slices, gate_of_row, add_dx, add_dh, add_dgate;
    int *status;
};

constexpr int kThreads = 256;

// Sums of K values over the block, the same in every thread.  `sh` is used by one round; the next round takes another.
template <int K>
__device__ __forceinline__ void block_sums(float (&v)[K], float (*sh)[32]) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) sh[k][threadIdx.x >> 5] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < kThreads / 32; ++q) t += sh[k][q];
        v[k] = t;
    }
}

// ---- rows that a block holds ------------------------------------------------------------------------------------------
// N values of a row for each of T threads, in pieces of one (SINGLES) or four (WHOLE: 16-byte accesses; the row is whole pieces
// at 16-byte addresses), the pieces of a thread T pieces apart.  The pieces that lie in the row are a thread's first `live` ones;
// the others are loaded as zeros and not stored.  FULL: whole pieces, and every thread has all of them.
enum Pieces { SINGLES, WHOLE, FULL };

template <int N, Pieces PIECES>
struct Row {
    static constexpr bool VEC = PIECES != SINGLES;
    static constexpr int W = VEC ? 4 : 1, P = N / W;
    int t, T, live;
    __device__ __forceinline__ Row(int t, int T, int width) : t(t), T(T) {
        const int last = (width + W - 1) / W - 1 - t;  // pieces behind this thread's first one
        live = last < 0 ? 0 : last / T + 1;
    }
    __device__ __forceinline__ bool in(int piece) const { return PIECES == FULL || piece < live; }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int i = 0; i < N; ++i) f(i);
    }
    // Takes a mean off, behind the row's end zeros stay.
    __device__ __forceinline__ void center(float (&v)[N], float mean) const {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = in(i / W) ? v[i] - mean : 0.f;
    }
    // First value of a piece.  Addresses are a row's own, the same in all threads, and this: a register for all arrays.
    __device__ __forceinline__ unsigned place(int piece) const { return unsigned(W) * unsigned(t + piece * T); }
    __device__ __forceinline__ void load(float (&v)[N], const float *row) const {
#pragma unroll
        for (int q = 0; q < P; ++q)
            if constexpr (VEC) {
                const float4 f = in(q) ? *reinterpret_cast<const float4 *>(row + place(q)) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
            } else {
                v[q] = in(q) ? row[place(q)] : 0.f;
            }
    }
    __device__ __forceinline__ void store(const float (&v)[N], float *row, bool add) const {
#pragma unroll
        for (int q = 0; q < P; ++q)
            if (in(q)) {
                if constexpr (VEC) {
                    float4 f = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                    float4 *at = reinterpret_cast<float4 *>(row + place(q));
                    if (add) {
                        const float4 old = *at;
                        f.x += old.x; f.y += old.y; f.z += old.z; f.w += old.w;
                    }
                    *at = f;
                } else {
                    row[place(q)] = add ? row[place(q)] + v[q] : v[q];
                }
            }
    }
};

// Asks the part of `width` values at `at` that is whole 16-byte units into L2, some rows ahead of its loads: these then wait for
// L2 and not for HBM, whatever the row's alignment.  (Copies of whole rows to shared memory ahead of their use took as long on
// the large shapes, longer on rows of 512 to 1024 values, and the shared memory from the loads of everything else.)
__device__ __forceinline__ void ask_ahead(const float *at, int width) {
    const uintptr_t begin = (reinterpret_cast<uintptr_t>(at) + 15) & ~uintptr_t(15);
    const uintptr_t end = reinterpret_cast<uintptr_t>(at + width) & ~uintptr_t(15);
    if (end > begin) prefetch_l2(reinterpret_cast<const void *>(begin), uint32_t(end - begin));
}

// The same for several arrays (null: none) by the first lanes of the row's warps, in turn.
template <int COUNT>
__device__ __forceinline__ void ask_all_ahead(const float *const (&arrays)[COUNT], size_t at, int width, int warp, int warps) {
    if ((threadIdx.x & 31) != 0) return;
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
        if (i % warps == warp && arrays[i] != nullptr) ask_ahead(arrays[i] + at, width);
}

constexpr int kMostThreads = 512;
constexpr int kNarrow = 4;  // values a thread of narrow rows and of rows taken one value at a time

// Sums over the threads of a row; WARP: the row is a warp's.  Rounds take the two sets of places in turn: a thread that
// writes to a set again has passed the barrier of the round between, and so have that set's readers.
//
// Up to four sums share one butterfly: each step halves the lanes that carry a sum instead of repeating itself for every sum,
// 6 exchanges for four sums instead of 20 (with those, and every thread adding up all warps' sums, the two rounds were half of
// the backward's 890 instructions a row and warp, which bound it: 207 us at 16384 x 2048).
template <int K>
__device__ __forceinline__ float packed_sum(const float (&v)[K]) {  // of v[lane / (32 / K)], over the lanes
    static_assert(K == 1 || K == 2 || K == 4, "sums to a round");
    const int lane = threadIdx.x & 31;
    float x;
    if constexpr (K == 4) {
        const bool high = lane & 16, odd = lane & 8;
        const float a = (high ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, high ? v[0] : v[2], 16);
        const float b = (high ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, high ? v[1] : v[3], 16);
        x = (odd ? b : a) + __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
    } else if constexpr (K == 2) {
        const bool high = lane & 16;
        x = (high ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, high ? v[0] : v[1], 16);
    } else {
        x = v[0];
    }
#pragma unroll
    for (int o = 16 / K; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

using Places = float[2][4][32];  // sums of up to 32 warps, zeros where there are fewer

__device__ __forceinline__ void clear_places(Places &places) {
    if (threadIdx.x < 32)
#pragma unroll
        for (int i = 0; i < 8; ++i) places[i >> 2][i & 3][threadIdx.x] = 0.f;
}

template <bool WARP>
struct Rounds {
    Places &places;
    int turn;
    template <int K>
    __device__ __forceinline__ void sums(float (&v)[K]) {
        constexpr int L = 32 / K;  // lanes to a sum
        float x = packed_sum(v);
        const int lane = threadIdx.x & 31;
        if (!WARP) {
            if (lane % L == 0) places[turn][lane / L][threadIdx.x >> 5] = x;
            __syncthreads();
            x = 0.f;
#pragma unroll
            for (int q = 0; q < kMostThreads / 32; q += L) x += places[turn][lane / L][q + lane % L];
#pragma unroll
            for (int o = (L < 16 ? L : 16) / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            turn ^= 1;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = __shfl_sync(0xffffffffu, x, k * L);
    }
};

template <int N, Pieces PIECES, bool WARP, bool LAYER>
__global__ void __launch_bounds__(kMostThreads, N == kNarrow ? 2 : 1) norm_fwd_kernel(const __grid_constant__ Forward p) {
    __shared__ Places places;
    launch_next();
    if (!WARP) {
        clear_places(places);
        __syncthreads();
    }
    launch_wait();
    Rounds<WARP> rounds = {places, 0};
    const Row<N, PIECES> row_of(WARP ? threadIdx.x & 31 : threadIdx.x, WARP ? 32 : blockDim.x, p.cols);
    const unsigned per_block = WARP ? blockDim.x >> 5 : 1;
    const float inv = 1.f / float(p.cols);
    const bool gate_each = p.gate && p.rows_per_gate == 1;
    unsigned long long row = (unsigned long long)blockIdx.x * per_block + (WARP ? threadIdx.x >> 5 : 0);
    const unsigned long long step = (unsigned long long)gridDim.x * per_block;
    const float *const ahead[3] = {p.x, p.h, gate_each ? p.gate : nullptr};
    for (; row < p.rows; row += step) {
        const size_t at = row * size_t(p.cols);
        float v[N], u[N], w[N];
        row_of.load(v, p.x + at);
        if (p.ahead && row + step < p.rows) ask_all_ahead(ahead, (row + step) * size_t(p.cols), p.cols, WARP ? 0 : threadIdx.x >> 5, WARP ? 1 : blockDim.x >> 5);
        if (p.h) {
            row_of.load(u, p.h + at);
            float g[N];
            if (p.gate) row_of.load(g, p.gate + (gate_each ? at : row / p.rows_per_gate * p.cols));
            if (p.post_w) {
                float m[1] = {0.f}, sq[1] = {0.f};
                if (LAYER) {
                    row_of.each([&](int i) { m[0] += u[i]; });
                    rounds.sums(m);
                    row_of.center(u, m[0] * inv);
                }
                row_of.each([&](int i) { sq[0] += u[i] * u[i]; });
                row_of.load(w, p.post_w);
                rounds.sums(sq);
                const float rstd = rsqrtf(sq[0] * inv + p.eps);
                row_of.each([&](int i) { u[i] *= rstd * w[i]; });
                if (p.post_b) {
                    row_of.load(w, p.post_b);
                    row_of.each([&](int i) { u[i] += w[i]; });
                }
            }
            row_of.each([&](int i) { v[i] += p.scale * (p.gate ? g[i] * u[i] : u[i]); });
            row_of.store(v, p.r + at, false);
        }
        if (p.n) {
            float m[1] = {0.f}, sq[1] = {0.f};
            if (LAYER) {
                row_of.each([&](int i) { m[0] += v[i]; });
                rounds.sums(m);
                row_of.center(v, m[0] * inv);
            }
            row_of.each([&](int i) { sq[0] += v[i] * v[i]; });
            row_of.load(w, p.pre_w);
            rounds.sums(sq);
            const float rstd = rsqrtf(sq[0] * inv + p.eps);
            row_of.each([&](int i) { v[i] *= rstd * w[i]; });
            if (p.pre_b) {
                row_of.load(w, p.pre_b);
                row_of.each([&](int i) { v[i] += w[i]; });
            }
            row_of.store(v, p.n + at, false);
        }
    }
}

// First and last row of the block's share; a block has one piece of a group or several whole groups.
__device__ __forceinline__ void rows_of_block(const Backward &p, unsigned block, unsigned blocks, unsigned long long *begin, unsigned long long *end) {
    const unsigned long long length = p.rows / p.groups;
    if (p.slices > 1) {
        const unsigned long long group = block / p.slices, s = block % p.slices;
        *begin = group * length + length * s / p.slices;
        *end = group * length + length * (s + 1) / p.slices;
    } else {
        *begin = p.groups * block / blocks * length;
        *end = p.groups * (block + 1) / blocks * length;
    }
}

// What a backward kernel adds up: without biases a row takes fewer instructions and registers.
enum Sums { RMS, RMS_BIAS, LAYER_BIAS };

constexpr int kValues = 8;       // a thread's, in the backward
constexpr int kMostCluster = 4;  // blocks to a row

// Backward of rows that a block (or a cluster of blocks, each with a slab of `width` columns) holds, eight values a thread.  A
// thread keeps its columns' sums over the block's rows in registers.  What bounds it is the instructions of a row
// and its two rounds of sums, with 16 warps to an SM, beside the 2000 clocks that HBM takes for 2048 values on every SM (16384 x 2048:
// 143 us, layer norms 164, HBM 125).  On clusters an SM has one block and 37 to 41 % of its issue slots are used: the latencies of
// a row's loads and exchanges follow each other (2048 x 8192: 105 us, layer norms 144, HBM 62).
//
// Layer norms on clusters: the mean is each block's own at first, and the sums about it are moved to the row's mean when the
// blocks exchange them, so that a row has two exchanges like one of RMS norms and not three.
// Blocks of one warp have no barriers and no places to meet at (200000 x 64: 101 us, with them 131).
template <int N, int THREADS, Sums MODE, Pieces PIECES, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, (N == kNarrow ? 768 : kMostThreads) / THREADS) norm_bwd_kernel(const __grid_constant__ Backward p, int slab) {
    constexpr bool LAYER = MODE == LAYER_BIAS, BIAS = MODE != RMS;
    __shared__ Places places;
    __shared__ __align__(16) float exchange[2][kMostCluster][8];  // CLUSTER: the blocks' sums of a round
    __shared__ uint64_t arrived[2];
    const unsigned rank = CLUSTER ? cluster_ctarank() : 0;
    const unsigned blocks_a_row = CLUSTER ? unsigned(p.cols + slab - 1) / unsigned(slab) : 1;
    const int c0 = int(rank) * slab, width = CLUSTER ? min(slab, p.cols - c0) : p.cols;
    launch_next();
    if (THREADS > 32) {
        clear_places(places);
        __syncthreads();
    }
    if (CLUSTER) {
        if (threadIdx.x == 0) {
            mbar_init(&arrived[0], 1);
            mbar_init(&arrived[1], 1);
            mbar_init_fence();
        }
        cluster_sync_all();  // all blocks have begun and have their barriers: their shared memory may be written to
    }
    launch_wait();

    const Row<N, PIECES> row_of(threadIdx.x, blockDim.x, width);
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const float inv = 1.f / float(p.cols);
    const unsigned block = blockIdx.x / blocks_a_row, blocks = gridDim.x / blocks_a_row;
    const unsigned long long length = p.rows / p.groups;
    unsigned long long begin, end;
    rows_of_block(p, block, blocks, &begin, &end);
    const bool gate_each = p.gate && p.rows_per_gate == 1;
    const float *const ahead[5] = {p.r, p.h, p.dn, p.dr, gate_each ? p.gate : nullptr};

    Rounds<THREADS == 32> rounds = {places, 0};
    int turn = 0;
    // 4 * QUADS numbers of every block of the cluster, block q's at the result's [q]: a block writes its own to all.  The set of
    // places and barrier that a block writes to again are free: that block has had the exchange between, to which every block
    // came behind its reads.  (With cluster barriers, whose release waits for the row's stores, a row of 8192 took 1.6 times as
    // long.)
    int phase = 0;
    auto exchanged = [&](auto quads, const float4 &a, const float4 &b) -> const float (*)[8] {
        constexpr int QUADS = decltype(quads)::value;
        if (threadIdx.x == 0) mbar_arrive_expect_tx(&arrived[turn], blocks_a_row * QUADS * 16);
        if (threadIdx.x < blocks_a_row) {
            st_async_v4(&exchange[turn][rank][0], &arrived[turn], threadIdx.x, a);
            if (QUADS > 1) st_async_v4(&exchange[turn][rank][4], &arrived[turn], threadIdx.x, b);
        }
        mbar_wait_warp_cluster(&arrived[turn], phase, p.status, 191);
        const float (*const all)[8] = exchange[turn];
        phase ^= turn;
        turn ^= 1;
        return all;
    };
    const float count = float(slab), last_count = float(p.cols - int(blocks_a_row - 1) * slab);  // columns of the blocks
    using Quads = std::integral_constant<int, LAYER ? 2 : 1>;
    using Quad = std::integral_constant<int, 1>;

    float gate[N], sum_gate[N] = {}, sum_pre_w[N] = {}, sum_pre_b[N] = {}, sum_post_w[N] = {}, sum_post_b[N] = {};
    // rows until the gate's next row and until the end of the group that dgate is summed over
    unsigned long long gate_left = 0, group_left = begin < end ? length - begin % length : 0;
    size_t gate_at = 0;
    if (p.gate && !gate_each && begin < end) {
        const unsigned long long q = begin / p.rows_per_gate;
        gate_left = (q + 1) * p.rows_per_gate - begin;
        gate_at = q * p.cols + c0;
        row_of.load(gate, p.gate + gate_at);
    }
    size_t at = begin * size_t(p.cols) + c0;
    for (unsigned long long row = begin; row < end; ++row, at += p.cols) {
        float r[N], h[N], dn[N], dr[N], w[N];
        row_of.load(r, p.r + at);
        if (p.h) row_of.load(h, p.h + at);
        if (p.dn) row_of.load(dn, p.dn + at);
        if (p.dr) row_of.load(dr, p.dr + at);
        if (gate_each) {
            row_of.load(gate, p.gate + at);
        } else if (p.gate) {
            if (gate_left == 0) {
                gate_left = p.rows_per_gate;
                gate_at += p.cols;
                row_of.load(gate, p.gate + gate_at);
            }
            --gate_left;
        }
        if (row + 1 < end) ask_all_ahead(ahead, at + p.cols, width, warp, warps);
        float m[2] = {0.f, 0.f};  // means of r and h; on clusters this block's
        if (LAYER) {
            row_of.each([&](int i) { m[0] += r[i]; });
            if (p.post_w) row_of.each([&](int i) { m[1] += h[i]; });
            rounds.sums(m);
            const float own = CLUSTER ? 1.f / float(width) : inv;
            m[0] *= own;
            m[1] *= own;
            row_of.center(r, m[0]);
            if (p.post_w) row_of.center(h, m[1]);
        }
        float a[N], v[4] = {0.f, 0.f, 0.f, 0.f};  // squares of r and h, a (r - m) and a
        if (p.dn) {
            row_of.load(w, p.pre_w + c0);
            row_of.each([&](int i) {
                a[i] = dn[i] * w[i];
                v[0] += r[i] * r[i];
                v[2] += a[i] * r[i];
                if (LAYER) v[3] += a[i];
            });
        }
        if (p.post_w) row_of.each([&](int i) { v[1] += h[i] * h[i]; });
        rounds.sums(v);
        if (CLUSTER) {
            const float (*const all)[8] = exchanged(Quads(), make_float4(v[0], v[1], v[2], v[3]), make_float4(m[0], m[1], 0.f, 0.f));
            float mean[2] = {0.f, 0.f};
            if (LAYER) {
#pragma unroll
                for (unsigned q = 0; q < kMostCluster; ++q)
                    if (q < blocks_a_row) {
                        const float share = (q + 1 < blocks_a_row ? count : last_count) * inv;
                        const float2 own = *reinterpret_cast<const float2 *>(&all[q][4]);
                        mean[0] += share * own.x;
                        mean[1] += share * own.y;
                    }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = 0.f;
#pragma unroll
            for (unsigned q = 0; q < kMostCluster; ++q)
                if (q < blocks_a_row) {
                    const float4 sums = *reinterpret_cast<const float4 *>(&all[q][0]);
                    v[0] += sums.x;
                    v[1] += sums.y;
                    v[2] += sums.z;
                    v[3] += sums.w;
                    if (LAYER) {
                        const float n = q + 1 < blocks_a_row ? count : last_count;
                        const float2 own = *reinterpret_cast<const float2 *>(&all[q][4]);
                        const float d0 = own.x - mean[0], d1 = own.y - mean[1];
                        v[0] += n * d0 * d0;
                        v[1] += n * d1 * d1;
                        v[2] += d0 * sums.w;
                    }
                }
            if (LAYER) {
                row_of.center(r, mean[0] - m[0]);
                if (p.post_w) row_of.center(h, mean[1] - m[1]);
            }
        }
        if (!p.dr) row_of.each([&](int i) { dr[i] = 0.f; });
        if (p.dn) {
            const float rs = rsqrtf(v[0] * inv + p.eps), c_hat = v[2] * rs * inv, c_one = LAYER ? v[3] * inv : 0.f;
            row_of.each([&](int i) {
                const float hat = r[i] * rs;
                dr[i] += rs * (LAYER ? a[i] - hat * c_hat - c_one : a[i] - hat * c_hat);  // all of r's gradient from here on
                sum_pre_w[i] += dn[i] * hat;
                if (BIAS) sum_pre_b[i] += dn[i];
            });
        }
        if (p.dx) row_of.store(dr, p.dx + at, p.add_dx);
        if (!p.h) continue;
        float q[LAYER ? 2 : 1] = {}, b[N];  // b h^ and b behind the block
        const float hs = rsqrtf(v[1] * inv + p.eps);
        // gate times gradient; dr turns into the gate's gradient
        row_of.each([&](int i) {
            dr[i] *= p.scale;
            b[i] = p.gate ? gate[i] * dr[i] : dr[i];
        });
        if (p.post_w) {
            row_of.load(w, p.post_w + c0);
            row_of.each([&](int i) {
                h[i] *= hs;
                sum_post_w[i] += b[i] * h[i];
                if (BIAS) sum_post_b[i] += b[i];
                b[i] *= w[i];
                q[0] += b[i] * h[i];
                if constexpr (LAYER) q[1] += b[i];
            });
            if (p.gate) {
                if (BIAS && p.post_b) {
                    float bias[N];
                    row_of.load(bias, p.post_b + c0);
                    row_of.each([&](int i) { dr[i] *= h[i] * w[i] + bias[i]; });
                } else {
                    row_of.each([&](int i) { dr[i] *= h[i] * w[i]; });
                }
            }
        } else {
            row_of.each([&](int i) { dr[i] *= h[i]; });
        }
        if (p.gate_of_row) {
            row_of.store(dr, p.dgate + at, p.add_dgate);
        } else if (p.gate) {
            row_of.each([&](int i) { sum_gate[i] += dr[i]; });
            if (--group_left == 0 && p.dgate) {
                group_left = length;
                row_of.store(sum_gate, p.dgate + row / length * p.cols + c0, p.add_dgate);
                row_of.each([&](int i) { sum_gate[i] = 0.f; });
            }
        }
        if (!p.dh) continue;
        if (p.post_w) {
            rounds.sums(q);
            float q_hat = q[0], q_one = 0.f;
            if constexpr (LAYER) q_one = q[1];
            if (CLUSTER) {
                const float (*const all)[8] = exchanged(Quad(), make_float4(q_hat, q_one, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f));
                q_hat = q_one = 0.f;
#pragma unroll
                for (unsigned k = 0; k < kMostCluster; ++k)
                    if (k < blocks_a_row) {
                        const float2 sums = *reinterpret_cast<const float2 *>(&all[k][0]);
                        q_hat += sums.x;
                        q_one += sums.y;
                    }
            }
            q_hat *= inv;
            q_one *= inv;
            row_of.each([&](int i) { b[i] = hs * (LAYER ? b[i] - h[i] * q_hat - q_one : b[i] - h[i] * q_hat); });
        }
        row_of.store(b, p.dh + at, p.add_dh);
    }
    const size_t mine = size_t(block) * p.cols + c0;
    if (p.partial[DPRE_W]) row_of.store(sum_pre_w, p.partial[DPRE_W] + mine, false);
    if (BIAS && p.partial[DPRE_B]) row_of.store(sum_pre_b, p.partial[DPRE_B] + mine, false);
    if (p.partial[DPOST_W]) row_of.store(sum_post_w, p.partial[DPOST_W] + mine, false);
    if (BIAS && p.partial[DPOST_B]) row_of.store(sum_post_b, p.partial[DPOST_B] + mine, false);
    if (p.partial[DGATE]) row_of.store(sum_gate, p.partial[DGATE] + mine, false);
    if (CLUSTER) cluster_sync_all();  // no block leaves while another may still write to it
}

// ---- rows of any length: every round of sums reads its row again (from L2, mostly) ---------------------------------
// For rows that no block or cluster holds (forward: above 16384 values, 8192 where they are not whole pieces; backward: 16384 and 4096).
// One value an access, and in the backward each row adds to the sums in global memory.  Forward of 2000 x 10001: 195 us, layer
// norms 266 (HBM 50); backward of 2000 x 5003: 265 and 389 (HBM 37), of 1600 x 20000: 940 and 1306 (HBM 119).
template <bool LAYER>
__global__ void __launch_bounds__(kThreads) norm_fwd_long_kernel(const __grid_constant__ Forward p) {
    __shared__ float sh[4][1][32];
    launch_next();
    launch_wait();
    const float inv = 1.f / float(p.cols);
    for (unsigned long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const size_t at = row * size_t(p.cols);
        const float *x = p.x + at, *h = p.h ? p.h + at : nullptr, *gate = p.gate ? p.gate + row / p.rows_per_gate * p.cols : nullptr;
        float hm[1] = {0.f}, hs[1] = {0.f}, rm[1] = {0.f}, rs[1] = {0.f};
        if (p.post_w) {
            if (LAYER) {
                for (int j = threadIdx.x; j < p.cols; j += kThreads) hm[0] += h[j];
                block_sums(hm, sh[0]);
                hm[0] *= inv;
            }
            for (int j = threadIdx.x; j < p.cols; j += kThreads) hs[0] += (h[j] - hm[0]) * (h[j] - hm[0]);
            block_sums(hs, sh[1]);
            hs[0] = rsqrtf(hs[0] * inv + p.eps);
        }
        for (int j = threadIdx.x; j < p.cols; j += kThreads) {
            float v = x[j];
            if (h) {
                float u = h[j];
                if (p.post_w) u = (u - hm[0]) * hs[0] * p.post_w[j] + (p.post_b ? p.post_b[j] : 0.f);
                v += p.scale * (gate ? gate[j] * u : u);
                p.r[at + j] = v;
            }
            if (LAYER) rm[0] += v;
            else rs[0] += v * v;
        }
        if (p.n) {
            const float *r = h ? p.r + at : x;  // (a thread reads what it has written itself)
            if (LAYER) {
                block_sums(rm, sh[2]);
                rm[0] *= inv;
                for (int j = threadIdx.x; j < p.cols; j += kThreads) rs[0] += (r[j] - rm[0]) * (r[j] - rm[0]);
            }
            block_sums(rs, sh[3]);
            rs[0] = rsqrtf(rs[0] * inv + p.eps);
            for (int j = threadIdx.x; j < p.cols; j += kThreads)
                p.n[at + j] = (r[j] - rm[0]) * rs[0] * p.pre_w[j] + (p.pre_b ? p.pre_b[j] : 0.f);
        }
        __syncthreads();  // the next row's sums go to the same places
    }
}

template <bool LAYER>
__global__ void __launch_bounds__(kThreads) norm_bwd_long_kernel(const __grid_constant__ Backward p) {
    __shared__ float sh[2][32], sh4[4][32], sh2[2][32];
    launch_next();
    launch_wait();
    const float inv = 1.f / float(p.cols);
    const unsigned long long length = p.rows / p.groups;
    unsigned long long begin, end;
    rows_of_block(p, blockIdx.x, gridDim.x, &begin, &end);
    const size_t mine = size_t(blockIdx.x) * p.cols;
    auto add = [&](Sum s, int j, float v, bool first) {
        float *q = p.partial[s] + mine + j;
        *q = first ? v : *q + v;
    };
    if (begin >= end)
        for (int s = 0; s < SUMS; ++s)
            if (p.partial[s])
                for (int j = threadIdx.x; j < p.cols; j += kThreads) p.partial[s][mine + j] = 0.f;
    for (unsigned long long row = begin; row < end; ++row) {
        const size_t at = row * size_t(p.cols);
        const bool first = row == begin, first_of_group = row % length == 0;
        const float *r = p.r + at, *h = p.h ? p.h + at : nullptr, *dr = p.dr ? p.dr + at : nullptr, *dn = p.dn ? p.dn + at : nullptr;
        const float *gate = p.gate ? p.gate + row / p.rows_per_gate * p.cols : nullptr;
        float m[2] = {0.f, 0.f};  // means of r and h
        if (LAYER) {
            for (int j = threadIdx.x; j < p.cols; j += kThreads) {
                m[0] += r[j];
                if (p.post_w) m[1] += h[j];
            }
            block_sums(m, sh);
            m[0] *= inv;
            m[1] *= inv;
        }
        float v[4] = {0.f, 0.f, 0.f, 0.f};  // squares of r and h, a (r - m) and a
        for (int j = threadIdx.x; j < p.cols; j += kThreads) {
            if (dn) {
                const float d = r[j] - m[0], a = dn[j] * p.pre_w[j];
                v[0] += d * d;
                v[2] += a * d;
                v[3] += a;
            }
            if (p.post_w) v[1] += (h[j] - m[1]) * (h[j] - m[1]);
        }
        block_sums(v, sh4);
        const float rs = rsqrtf(v[0] * inv + p.eps), hs = rsqrtf(v[1] * inv + p.eps);
        const float c_hat = v[2] * rs * inv, c_one = LAYER ? v[3] * inv : 0.f;
        auto full = [&](int j, float *hat) {  // D, and r^
            float d = dr ? dr[j] : 0.f;
            if (dn) {
                *hat = (r[j] - m[0]) * rs;
                d += rs * (dn[j] * p.pre_w[j] - *hat * c_hat - c_one);
            }
            return d;
        };
        float q[2] = {0.f, 0.f};  // a h^ and a behind the block
        for (int j = threadIdx.x; j < p.cols; j += kThreads) {
            float hat = 0.f;
            const float d = full(j, &hat);
            if (p.dx) p.dx[at + j] = p.add_dx ? p.dx[at + j] + d : d;
            if (p.partial[DPRE_W]) add(DPRE_W, j, dn[j] * hat, first);
            if (p.partial[DPRE_B]) add(DPRE_B, j, dn[j], first);
            if (!h) continue;
            const float sd = p.scale * d, du = gate ? gate[j] * sd : sd;
            float u = h[j];
            if (p.post_w) {
                const float h_hat = (u - m[1]) * hs, a = du * p.post_w[j];
                q[0] += a * h_hat;
                q[1] += a;
                if (p.partial[DPOST_W]) add(DPOST_W, j, du * h_hat, first);
                if (p.partial[DPOST_B]) add(DPOST_B, j, du, first);
                u = h_hat * p.post_w[j] + (p.post_b ? p.post_b[j] : 0.f);
            } else if (p.dh) {
                p.dh[at + j] = p.add_dh ? p.dh[at + j] + du : du;
            }
            if (p.dgate) {
                float *o = p.dgate + (p.gate_of_row ? row : row / length) * p.cols + j;
                const float v = sd * u;
                *o = (p.gate_of_row || first_of_group) && !p.add_dgate ? v : *o + v;
            } else if (p.partial[DGATE]) {
                add(DGATE, j, sd * u, first);
            }
        }
        if (p.post_w && p.dh) {
            block_sums(q, sh2);
            q[0] *= inv;
            q[1] = LAYER ? q[1] * inv : 0.f;
            for (int j = threadIdx.x; j < p.cols; j += kThreads) {
                float hat = 0.f;
                const float sd = p.scale * full(j, &hat), du = gate ? gate[j] * sd : sd;
                const float o = hs * (du * p.post_w[j] - (h[j] - m[1]) * hs * q[0] - q[1]);
                p.dh[at + j] = p.add_dh ? p.dh[at + j] + o : o;
            }
        }
        __syncthreads();
    }
}

// ---- the blocks' sums, added up ------------------------------------------------------------------------------------
struct Fold {
    const float *partial;
    float *out;
    int parts, add;
    unsigned long long results;  // rows of the output; result i is the sum of parts i * parts .. + parts - 1
};

struct Folds {
    Fold f[SUMS];
    int cols, folds;
};

constexpr int kFoldThreads = 1024;  // 32 columns by 32 parts at a time
// Parts that are on their way together, also where fewer are left: one round for 300 blocks' sums (an unrolled loop takes its last
// ones one by one, each after the other's way to L2 and back: backward of 300 x 1024 9.5 us, 8.8 so).  Few parts are better off
// with that loop (30 x 10000: 10.9 us, 13.2 in batches).
constexpr int kFoldBatch = 10;

// Narrow rows leave few columns and many parts: clusters of SPLIT blocks share an item's parts, and the first block adds up what
// the others write into its shared memory (backward of 8000 x 128: 15 us, 26 with a block to an item).  The two sets of places take
// turns: a block that writes to a set again has passed the barrier of the item between, and so has that set's reader.
template <int SPLIT>
__global__ void __launch_bounds__(kFoldThreads, 2) norm_fold_kernel(const __grid_constant__ Folds p) {
    __shared__ float sh[32][33];
    __shared__ float sums[2][SPLIT][32];
    launch_next();
    if (SPLIT > 1) cluster_sync_all();  // all blocks have begun: their shared memory may be written to
    launch_wait();
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int rank = SPLIT > 1 ? int(cluster_ctarank()) : 0;
    const unsigned tiles = unsigned(p.cols + 31) / 32, step = gridDim.x / SPLIT;
    unsigned long long item = blockIdx.x / SPLIT;
    int turn = 0;
    for (int k = 0; k < p.folds; ++k) {
        const Fold &f = p.f[k];
        for (; item < f.results * tiles; item += step) {
            const unsigned long long result = item / tiles;
            const int col = int(item - result * tiles) * 32 + lane;
            const float *src = f.partial + result * f.parts * p.cols;
            float s = 0.f;
            if (col < p.cols && f.parts > 96 * SPLIT) {
                for (int q = 32 * rank + part; q < f.parts; q += 32 * SPLIT * kFoldBatch) {
                    float v[kFoldBatch];
#pragma unroll
                    for (int i = 0; i < kFoldBatch; ++i) {
                        const int at = q + 32 * SPLIT * i;
                        v[i] = at < f.parts ? __ldcg(src + size_t(at) * p.cols + col) : 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < kFoldBatch; ++i) s += v[i];
                }
            } else if (col < p.cols) {
                for (int q = 32 * rank + part; q < f.parts; q += 32 * SPLIT) s += __ldcg(src + size_t(q) * p.cols + col);
            }
            sh[part][lane] = s;
            __syncthreads();
            // warp `part` adds up column `part` of the tile
            float t = sh[lane][part];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            const int mine = int(item - result * tiles) * 32 + part;
            if (SPLIT > 1) {
                if (lane == 0) st_cluster(map_to_rank(&sums[turn][rank][part], 0), t);
                __syncwarp();
                cluster_sync_all();
                t = 0.f;
#pragma unroll
                for (int q = 0; q < SPLIT; ++q) t += sums[turn][q][part];
                turn ^= 1;
            }
            if (lane == 0 && rank == 0 && mine < p.cols) {
                float *o = f.out + result * p.cols + mine;
                *o = f.add ? *o + t : t;
            }
            __syncthreads();
        }
        item -= f.results * tiles;
    }
}

template <typename... Params, typename... Args>
int32_t start(katsu_cuda_ctx *ctx, void (*kernel)(Params...), unsigned grid, unsigned block, Args &&...args) {
    return katsu_launch_chained(ctx, kernel, grid, block, 0, 1, args...);
}

// Blocks to an SM, by the registers of the kernels that hold rows (up to 128 a thread).
unsigned resident_blocks(unsigned threads) { return 512 / threads; }

// Whether rows are whole 16-byte pieces at 16-byte addresses.
bool pieces(int cols, std::initializer_list<const void *> pointers) {
    uintptr_t at = uintptr_t(cols) * sizeof(float);
    for (const void *q : pointers) at |= reinterpret_cast<uintptr_t>(q);
    return (at & 15u) == 0;
}

template <bool LAYER>
int32_t start_forward(katsu_cuda_ctx *ctx, Forward p) {
    const bool vec = pieces(p.cols, {p.x, p.h, p.gate, p.post_w, p.post_b, p.pre_w, p.pre_b, p.r, p.n});
    const unsigned long long sms = ctx->num_sms;
    if (p.cols > kMostThreads * (vec ? 32 : 16))
        return start(ctx, norm_fwd_long_kernel<LAYER>, unsigned(p.rows < sms * 4 ? p.rows : sms * 4), kThreads, p);
    // 16 values a thread, 32 where that would take more than 512 threads; up to 512 values are one warp's.  Four a thread, with
    // twice the warps to an SM, for rows of up to 128 values (65536 x 128: 26 us, with sixteen a thread 36) and rows of up to 2048
    // that go one value at a time (4000 x 1367, layer norms: 37 us, with sixteen 42).
    const bool wide = p.cols > kMostThreads * 16, narrow = p.cols <= (vec ? 32 : kMostThreads) * kNarrow, warp = p.cols <= (narrow ? 32 * kNarrow : 512);
    const unsigned threads = warp ? 128 : unsigned(katsu_div_up(katsu_div_up(p.cols, wide ? 32 : narrow ? kNarrow : 16), 32)) * 32;
    const unsigned long long need = warp ? katsu_div_up(p.rows, 4) : p.rows, most = sms * (narrow ? 1024 / threads : resident_blocks(threads));
    // Rows are asked into L2 ahead where little else of the SM runs under a row's rounds: layer norms have two more of them
    // (16384 x 2048: 90 us, 103 without), rows of more than 4096 values leave an SM to one block (8192 x 5120: 108 us, 127).  Two
    // blocks of RMS norms reach 93 % of HBM's rate without and 87 % with it.
    p.ahead = !warp && (LAYER || (threads > 256 && !wide));
    auto kernel = wide     ? norm_fwd_kernel<32, WHOLE, false, LAYER>
                  : narrow ? (vec ? norm_fwd_kernel<kNarrow, WHOLE, true, LAYER>
                               : warp ? norm_fwd_kernel<kNarrow, SINGLES, true, LAYER> : norm_fwd_kernel<kNarrow, SINGLES, false, LAYER>)
                  : warp ? norm_fwd_kernel<16, WHOLE, true, LAYER>  // (single values: narrow)
                         : (vec ? norm_fwd_kernel<16, WHOLE, false, LAYER> : norm_fwd_kernel<16, SINGLES, false, LAYER>);
    return start(ctx, kernel, unsigned(need < most ? need : most), threads, p);
}

// How the kernels' blocks share a row, and how many rows are on their way at once.
struct BackwardShape {
    int slab;  // columns to a block; 0: the kernel for rows of any length
    Pieces pieces;
    unsigned threads, cluster;
    bool narrow;
    size_t most_blocks;
};

BackwardShape backward_shape(const katsu_cuda_ctx *ctx, const Backward &p, std::initializer_list<const void *> pointers) {
    BackwardShape s = {};
    const int most = kMostThreads * kValues;  // columns to a block
    const bool vec = pieces(p.cols, pointers);
    if (p.cols > (vec ? kMostCluster * most : most)) {
        s.most_blocks = size_t(ctx->num_sms) * 4;
        return s;
    }
    s.cluster = p.cols > 2 * most ? 4 : p.cols > most ? 2 : 1;
    // Four values a thread as in the forward, here with half as many warps again to an SM: 65536 x 128 45 us, with eight a thread
    // 51; 4000 x 1367, layer norms, 69 and 81.
    s.narrow = p.cols <= (vec ? 32 : 384) * kNarrow;
    s.slab = int(katsu_div_up(katsu_div_up(p.cols, s.cluster), 4)) * 4;
    s.threads = unsigned(katsu_div_up(katsu_div_up(s.slab, s.narrow ? kNarrow : kValues), 32)) * 32;
    s.pieces = !vec ? SINGLES : p.cols == int(s.cluster * s.threads) * kValues ? FULL : WHOLE;
    s.most_blocks = size_t(ctx->num_sms) * (s.narrow ? 768 / s.threads : resident_blocks(s.threads)) / s.cluster;
    return s;
}

using BackwardKernel = void (*)(Backward, int);

template <Sums MODE>
BackwardKernel backward_of(const BackwardShape &s) {
    constexpr int most = kMostThreads;
    if (s.cluster > 1) return s.pieces == FULL ? norm_bwd_kernel<kValues, most, MODE, FULL, true> : norm_bwd_kernel<kValues, most, MODE, WHOLE, true>;
    if (s.narrow && s.threads == 32)
        return s.pieces == SINGLES ? norm_bwd_kernel<kNarrow, 32, MODE, SINGLES, false> : norm_bwd_kernel<kNarrow, 32, MODE, WHOLE, false>;
    if (s.narrow) return norm_bwd_kernel<kNarrow, 384, MODE, SINGLES, false>;
    if (s.threads == 32) return norm_bwd_kernel<kValues, 32, MODE, WHOLE, false>;
    return s.pieces == FULL    ? norm_bwd_kernel<kValues, most, MODE, FULL, false>
           : s.pieces == WHOLE ? norm_bwd_kernel<kValues, most, MODE, WHOLE, false> : norm_bwd_kernel<kValues, most, MODE, SINGLES, false>;
}

// Blocks (clusters) that go round at once.  Four SMs of a cluster are of one group of SMs, whose number four need not divide: 33
// clusters of 512 threads a block, where 148 SMs would have 37, and the last four took as long as the others before them
// (2048 x 16384, without gate and norm behind the block: 252 us, 33 clusters 149).
int32_t blocks_at_once(const katsu_cuda_ctx *ctx, BackwardKernel kernel, const BackwardShape &s, size_t *blocks) {
    *blocks = s.most_blocks;
    if (s.cluster <= 2) return KATSU_OK;
    cudaLaunchAttribute of_cluster = {};
    of_cluster.id = cudaLaunchAttributeClusterDimension;
    of_cluster.val.clusterDim.x = s.cluster;
    of_cluster.val.clusterDim.y = of_cluster.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(s.most_blocks) * s.cluster, 1, 1);
    config.blockDim = dim3(s.threads, 1, 1);
    config.attrs = &of_cluster;
    config.numAttrs = 1;
    int most = 0;
    KATSU_CUDA_TRY(cudaOccupancyMaxActiveClusters(&most, kernel, &config));
    if (most >= 1 && size_t(most) < *blocks) *blocks = size_t(most);
    return KATSU_OK;
}

struct Extent {
    const float *at;
    size_t bytes;
};

bool overlap(const Extent &a, const Extent &b) { return katsu_overlap(a.at, a.bytes, b.at, b.bytes); }

int32_t check_sizes(size_t rows, size_t cols, const float *gate, size_t gate_rows, int32_t kind, float eps) {
    KATSU_REQUIRE(kind == KATSU_NORM_RMS || kind == KATSU_NORM_LAYER, "unknown kind of norm");
    KATSU_REQUIRE(eps >= 0.f && eps < INFINITY, "eps must be 0 or more, and finite");
    KATSU_REQUIRE(cols >= 1 && cols <= 0x3fffffff, "rows must have 1 to 2^30 - 1 values");
    KATSU_REQUIRE(rows <= (size_t(1) << 62) / 4 / cols, "too many rows");
    KATSU_REQUIRE((gate != nullptr) == (gate_rows != 0), "gate and gate_rows go together");
    KATSU_REQUIRE(gate == nullptr || rows % gate_rows == 0, "gate_rows must divide rows");
    return KATSU_OK;
}

}  // namespace

extern "C" int32_t katsu_cuda_block_norm_fwd(katsu_cuda_ctx *ctx, const float *x, const float *h, const float *gate,
                                             size_t gate_rows, const float *post_w, const float *post_b,
                                             const float *pre_w, const float *pre_b, float scale, float eps, int32_t kind,
                                             float *r, float *n, size_t rows, size_t cols) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_TRY(check_sizes(rows, cols, gate, gate_rows, kind, eps));
    KATSU_REQUIRE(h != nullptr || (!gate && !post_w && !r), "without h there is no gate, no norm behind it and no sum");
    KATSU_REQUIRE(post_w != nullptr || !post_b, "a bias without weights");
    KATSU_REQUIRE((pre_w != nullptr) == (n != nullptr), "n and pre_w go together");
    KATSU_REQUIRE(pre_w != nullptr || !pre_b, "a bias without weights");
    KATSU_REQUIRE((h != nullptr) == (r != nullptr) && (r || n), "nothing to compute, or h without r");
    if (rows == 0) return katsu_bind(ctx);
    KATSU_REQUIRE(x != nullptr, "x is null");
    const size_t all = rows * cols * sizeof(float), channels = cols * sizeof(float), gates = gate_rows * channels;
    const Extent ins[] = {{x, all}, {h, all}, {gate, gates}, {post_w, channels}, {post_b, channels}, {pre_w, channels}, {pre_b, channels}};
    for (const Extent &in : ins)
        KATSU_REQUIRE(!overlap(in, {r, all}) && !overlap(in, {n, all}), "an output is an input too, or overlaps one");
    KATSU_REQUIRE(!overlap({r, all}, {n, all}), "r and n are the same buffer, or overlap");
    KATSU_TRY(katsu_bind(ctx));
    Forward p = {x, h, gate, post_w, post_b, pre_w, pre_b, r, n, scale, eps, rows, gate ? rows / gate_rows : 1, (int)cols, 0};
    return kind == KATSU_NORM_LAYER ? start_forward<true>(ctx, p) : start_forward<false>(ctx, p);
}

extern "C" int32_t katsu_cuda_block_norm_bwd(katsu_cuda_ctx *ctx, const float *r, const float *h, const float *gate,
                                             size_t gate_rows, const float *post_w, const float *post_b,
                                             const float *pre_w, float scale, float eps, int32_t kind, const float *dr,
                                             const float *dn, float *dx, float *dh, float *dgate, float *dpost_w,
                                             float *dpost_b, float *dpre_w, float *dpre_b, size_t rows, size_t cols,
                                             int32_t accumulate) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_TRY(check_sizes(rows, cols, gate, gate_rows, kind, eps));
    KATSU_REQUIRE(accumulate >= 0 && accumulate < 128, "unknown bits in accumulate");
    KATSU_REQUIRE(h != nullptr || (!gate && !post_w && !dh), "without h there is no gate, no norm behind it and no dh");
    KATSU_REQUIRE(post_w != nullptr || (!post_b && !dpost_w && !dpost_b), "post_b, dpost_w or dpost_b without post_w");
    KATSU_REQUIRE(gate != nullptr || !dgate, "dgate without a gate");
    KATSU_REQUIRE((pre_w != nullptr) == (dn != nullptr) || rows == 0, "dn and pre_w go together");
    KATSU_REQUIRE(pre_w != nullptr || (!dpre_w && !dpre_b), "dpre_w or dpre_b without pre_w");
    const size_t all = rows * cols * sizeof(float), channels = cols * sizeof(float), gates = gate_rows * channels;
    const Extent outs[] = {{dx, all}, {dh, all}, {dgate, gates}, {dpost_w, channels}, {dpost_b, channels}, {dpre_w, channels}, {dpre_b, channels}};
    const Extent ins[] = {{r, all}, {h, all}, {gate, gates}, {post_w, channels}, {post_b, channels}, {pre_w, channels}, {dr, all}, {dn, all}};
    for (size_t i = 0; i < 7; ++i) {
        for (size_t j = 0; j < i; ++j) KATSU_REQUIRE(!overlap(outs[i], outs[j]), "two outputs are the same buffer, or overlap");
        for (const Extent &in : ins) KATSU_REQUIRE(!overlap(in, outs[i]), "an output is an input too, or overlaps one");
    }
    const int adds[SUMS] = {accumulate & KATSU_BLOCK_DPRE_W, accumulate & KATSU_BLOCK_DPRE_B, accumulate & KATSU_BLOCK_DPOST_W,
                            accumulate & KATSU_BLOCK_DPOST_B, accumulate & KATSU_BLOCK_DGATE};
    float *const sums[SUMS] = {dpre_w, dpre_b, dpost_w, dpost_b, dgate};
    KATSU_REQUIRE(r != nullptr || rows == 0, "r is null");
    KATSU_TRY(katsu_bind(ctx));
    if (rows == 0) {
        for (int s = 0; s < DGATE; ++s)
            if (sums[s] && !adds[s]) KATSU_CUDA_TRY(cudaMemsetAsync(sums[s], 0, cols * sizeof(float), ctx->stream));
        if (dgate && !adds[DGATE]) KATSU_CUDA_TRY(cudaMemsetAsync(dgate, 0, gate_rows * cols * sizeof(float), ctx->stream));
        return KATSU_OK;
    }
    Backward p = {};
    p.r = r; p.h = h; p.gate = gate; p.post_w = post_w; p.post_b = post_b; p.pre_w = pre_w; p.dr = dr; p.dn = dn;
    p.dx = dx; p.dh = dh;
    p.scale = scale; p.eps = eps;
    p.rows = rows; p.rows_per_gate = gate ? rows / gate_rows : 1; p.cols = (int)cols;
    p.status = ctx->status;
    p.add_dx = accumulate & KATSU_BLOCK_DX; p.add_dh = accumulate & KATSU_BLOCK_DH; p.add_dgate = adds[DGATE];
    p.gate_of_row = dgate && gate_rows == rows;
    p.groups = dgate && !p.gate_of_row ? gate_rows : 1;
    const BackwardShape shape = backward_shape(ctx, p, {r, h, gate, post_w, post_b, pre_w, dr, dn, dx, dh, dgate});
    const bool layer = kind == KATSU_NORM_LAYER, bias = post_b || dpre_b || dpost_b;
    const BackwardKernel kernel = layer ? backward_of<LAYER_BIAS>(shape) : bias ? backward_of<RMS_BIAS>(shape) : backward_of<RMS>(shape);
    size_t want = 0;
    KATSU_TRY(blocks_at_once(ctx, kernel, shape, &want));
    if (want > rows) want = rows;
    size_t blocks;
    if (p.gate_of_row || dgate == nullptr || p.groups < want) {
        p.slices = (int)(want / p.groups);  // (a block more than go round at once would double the time)
        const size_t length = rows / p.groups;
        if ((size_t)p.slices > length) p.slices = (int)length;
        blocks = p.groups * p.slices;
    } else {
        p.slices = 1;
        blocks = want;
    }
    const bool gate_parts = dgate && !p.gate_of_row && p.slices > 1;
    if (dgate && !gate_parts) p.dgate = dgate;
    Folds folds = {};
    folds.cols = (int)cols;
    int parts = 0;
    for (int s = 0; s < SUMS; ++s) parts += s == DGATE ? gate_parts : sums[s] != nullptr;
    if (parts) {
        float *scratch = nullptr;
        KATSU_TRY(katsu_scratch(ctx, size_t(parts) * blocks * cols, &scratch));
        for (int s = 0; s < SUMS; ++s) {
            if (s == DGATE ? !gate_parts : sums[s] == nullptr) continue;
            p.partial[s] = scratch;
            folds.f[folds.folds++] = {scratch, sums[s], s == DGATE ? p.slices : (int)blocks, adds[s], s == DGATE ? p.groups : 1};
            scratch += blocks * cols;
        }
    }
    if (shape.slab == 0)
        KATSU_TRY(start(ctx, layer ? norm_bwd_long_kernel<true> : norm_bwd_long_kernel<false>, (unsigned)blocks, kThreads, p));
    else
        KATSU_TRY(katsu_launch_chained(ctx, kernel, (unsigned)blocks * shape.cluster, shape.threads, 0, shape.cluster, p, shape.slab));
    if (folds.folds == 0) return KATSU_OK;
    unsigned long long items = 0;
    for (int k = 0; k < folds.folds; ++k) items += folds.f[k].results * katsu_div_up(cols, 32);
    const unsigned long long most = (unsigned long long)ctx->num_sms * 2;
    const unsigned grid = unsigned(items < most ? items : most);
    // (24 clusters of eight are resident at once)
    if (blocks >= 512 && items <= 24) return katsu_launch_chained(ctx, norm_fold_kernel<8>, grid * 8, kFoldThreads, 0, 8, folds);
    if (blocks >= 512 && items <= 48) return katsu_launch_chained(ctx, norm_fold_kernel<4>, grid * 4, kFoldThreads, 0, 4, folds);
    return start(ctx, norm_fold_kernel<1>, grid, kFoldThreads, folds);
}
