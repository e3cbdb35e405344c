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
// A row belongs to one block.  Sums over rows (weights, biases, gate) are kept a block and folded by a second launch in a
// fixed order.  Variances are of differences from the mean, in a round of their own: mean(v^2) - m^2 in 32 bits would lose a
// row whose mean is a thousand times its spread.
#include <math.h>

#include <initializer_list>

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
    int cols;
    int *status;
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
template <int K, int T>
__device__ __forceinline__ void block_sums(float (&v)[K], float (*sh)[32]) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (T == 32) return;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) sh[k][threadIdx.x >> 5] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < T / 32; ++q) t += sh[k][q];
        v[k] = t;
    }
}

// ---- rows that a block holds ------------------------------------------------------------------------------------------
// N values of a row for each of T threads, in pieces of four (VEC: 16-byte accesses; the row is whole pieces at 16-byte
// addresses) or one, the pieces of a thread T pieces apart.  The pieces that lie in the row are a thread's first `live` ones;
// the others are loaded as zeros and not stored.
template <int N, bool VEC>
struct Row {
    static constexpr int W = VEC ? 4 : 1, P = N / W;
    int t, T, live;
    __device__ __forceinline__ Row(int t, int T, int width) : t(t), T(T) {
        const int last = (width + W - 1) / W - 1 - t;  // pieces behind this thread's first one
        live = last < 0 ? 0 : last / T + 1;
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int i = 0; i < N; ++i) f(i);
    }
    // Takes a row's mean off, behind whose end zeros stay.
    __device__ __forceinline__ void center(float (&v)[N], float mean) const {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i / W < live ? v[i] - mean : 0.f;
    }
    __device__ __forceinline__ void load(float (&v)[N], const float *at) const {
        at += W * t;
#pragma unroll
        for (int q = 0; q < P; ++q, at += W * T)
            if constexpr (VEC) {
                const float4 f = q < live ? *reinterpret_cast<const float4 *>(at) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
            } else {
                v[q] = q < live ? *at : 0.f;
            }
    }
    __device__ __forceinline__ void store(const float (&v)[N], float *at, bool add) const {
        at += W * t;
#pragma unroll
        for (int q = 0; q < P; ++q, at += W * T)
            if (q < live) {
                if constexpr (VEC) {
                    float4 f = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                    if (add) {
                        const float4 old = *reinterpret_cast<const float4 *>(at);
                        f.x += old.x; f.y += old.y; f.z += old.z; f.w += old.w;
                    }
                    *reinterpret_cast<float4 *>(at) = f;
                } else {
                    *at = add ? *at + v[q] : v[q];
                }
            }
    }
};

// Rows brought to shared memory ahead of their use: `arrays` arrays of `width` columns a row, `stages` rows.
struct Slab {
    int width, arrays, stages;
};

struct Ring {
    float *data;
    uint64_t *full;
    Slab slab;
    int stage, phase;  // of the row that is read next
    __device__ __forceinline__ void init(float *at, uint64_t *bars, const Slab &s) {
        data = at;
        full = bars;
        slab = s;
        stage = phase = 0;
        if (threadIdx.x == 0) {
            for (int i = 0; i < s.stages; ++i) mbar_init(&full[i], 1);
            mbar_init_fence();
        }
    }
    __device__ __forceinline__ const float *next(int *status) const {  // waits for the next row
        // (a wait that gives up leaves wrong values behind, which the next synchronising call reports)
        mbar_wait_warp_ready(&full[stage], phase, status, 191);
        return data + size_t(stage) * slab.arrays * slab.width;
    }
    __device__ __forceinline__ void advance() {
        if (++stage == slab.stages) {
            stage = 0;
            phase ^= 1;
        }
    }
    // By one thread: copies `width` columns of every array that there is, from `at` values behind its start, to a stage.
    __device__ __forceinline__ void fetch(int to_stage, std::initializer_list<const float *> arrays, size_t at, int width) const {
        const uint32_t bytes = uint32_t(width) * 4;
        float *to = data + size_t(to_stage) * slab.arrays * slab.width;
        mbar_arrive_expect_tx(&full[to_stage], bytes * slab.arrays);
        for (const float *src : arrays)
            if (src) {
                bulk_load(to, src + at, bytes, &full[to_stage]);
                to += slab.width;
            }
    }
};

constexpr int kMostStages = 8;
constexpr size_t kRoom = size_t(222) * 1024;  // shared memory of an SM for rings, less 2 KiB a block

constexpr int kMostThreads = 512;

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

// The ring leaves little of the SM's memory to L1, so what every row needs is kept beside it: a copy of `width` weights, if
// there are any, in shared memory at `to`, which moves behind it.
template <bool VEC>
__device__ __forceinline__ const float *keep_weights(const float *weights, float *&to, int width) {
    const float *copy = to;
    if (weights != nullptr) {
        if (VEC) {
            for (int j = 4 * threadIdx.x; j < width; j += 4 * blockDim.x)
                *reinterpret_cast<float4 *>(to + j) = __ldg(reinterpret_cast<const float4 *>(weights + j));
        } else {
            for (int j = threadIdx.x; j < width; j += blockDim.x) to[j] = __ldg(weights + j);
        }
        to += width;
    }
    return copy;
}

// How a row's threads find each other and its values: a warp's own row, a block's by plain loads, a block's by the ring.
enum Rows { OF_WARP, OF_BLOCK, BY_RING };

template <int N, bool VEC, Rows ROWS, bool LAYER>
__global__ void __launch_bounds__(kMostThreads) norm_fwd_kernel(const __grid_constant__ Forward p, const __grid_constant__ Slab slab) {
    constexpr bool WARP = ROWS == OF_WARP, RING = ROWS == BY_RING;
    extern __shared__ __align__(128) float ring_data[];
    __shared__ Places places;
    __shared__ uint64_t full[kMostStages];
    Ring ring;
    launch_next();
    if (RING) ring.init(ring_data, full, slab);
    if (!WARP) {
        clear_places(places);
        __syncthreads();
    }
    launch_wait();
    Rounds<WARP> rounds = {places, 0};
    const Row<N, VEC> row_of(WARP ? threadIdx.x & 31 : threadIdx.x, WARP ? 32 : blockDim.x, p.cols);
    const unsigned per_block = WARP ? blockDim.x >> 5 : 1;
    const float inv = 1.f / float(p.cols);
    const bool gate_each = p.gate && p.rows_per_gate == 1;
    unsigned long long row = (unsigned long long)blockIdx.x * per_block + (WARP ? threadIdx.x >> 5 : 0);
    const unsigned long long step = (unsigned long long)gridDim.x * per_block;
    float *keep_at = ring_data + (RING ? size_t(slab.stages) * slab.arrays * slab.width : 0);
    const float *post_w = RING ? keep_weights<VEC>(p.post_w, keep_at, p.cols) : p.post_w;
    const float *post_b = RING ? keep_weights<VEC>(p.post_b, keep_at, p.cols) : p.post_b;
    const float *pre_w = RING ? keep_weights<VEC>(p.pre_w, keep_at, p.cols) : p.pre_w;
    const float *pre_b = RING ? keep_weights<VEC>(p.pre_b, keep_at, p.cols) : p.pre_b;
    if (RING) __syncthreads();
    auto fetch = [&](int stage, unsigned long long r) {
        ring.fetch(stage, {p.x, p.h, gate_each ? p.gate : nullptr}, r * size_t(p.cols), p.cols);
    };
    if (RING && threadIdx.x == 0)
        for (int i = 0; i < slab.stages && row + i * step < p.rows; ++i) fetch(i, row + i * step);
    for (; row < p.rows; row += step) {
        const size_t at = row * size_t(p.cols);
        float v[N], u[N], w[N];
        const float *from = nullptr;
        bool refill = RING;  // behind the row's first barrier
        if (RING) from = ring.next(p.status);
        auto refilled = [&] {
            if (!RING || !refill) return;
            refill = false;
            if (threadIdx.x == 0 && row + slab.stages * step < p.rows) fetch(ring.stage, row + slab.stages * step);
            ring.advance();
        };
        row_of.load(v, RING ? from : p.x + at);
        if (p.h) {
            row_of.load(u, RING ? from + slab.width : p.h + at);
            float g[N];
            if (p.gate)
                row_of.load(g, RING && gate_each ? from + 2 * slab.width
                                                 : p.gate + (gate_each ? at : row / p.rows_per_gate * p.cols));
            if (RING) fence_proxy_async_smem();  // in front of the copies behind the first barrier
            if (p.post_w) {
                float m[1] = {0.f}, sq[1] = {0.f};
                if (LAYER) {
                    row_of.each([&](int i) { m[0] += u[i]; });
                    rounds.sums(m);
                    refilled();
                    m[0] *= inv;
                }
                if (LAYER) row_of.center(u, m[0]);
                row_of.each([&](int i) { sq[0] += u[i] * u[i]; });
                row_of.load(w, post_w);
                rounds.sums(sq);
                refilled();
                const float rstd = 1.f / sqrtf(sq[0] * inv + p.eps);
                row_of.each([&](int i) { u[i] *= rstd * w[i]; });
                if (p.post_b) {
                    row_of.load(w, post_b);
                    row_of.each([&](int i) { u[i] += w[i]; });
                }
            }
            row_of.each([&](int i) { v[i] += p.scale * (p.gate ? g[i] * u[i] : u[i]); });
            row_of.store(v, p.r + at, false);
        } else if (RING) {
            fence_proxy_async_smem();
        }
        if (p.n) {
            float m[1] = {0.f}, sq[1] = {0.f};
            if (LAYER) {
                row_of.each([&](int i) { m[0] += v[i]; });
                rounds.sums(m);
                refilled();
                m[0] *= inv;
            }
            if (LAYER) row_of.center(v, m[0]);
            row_of.each([&](int i) { sq[0] += v[i] * v[i]; });
            row_of.load(w, pre_w);
            rounds.sums(sq);
            refilled();
            const float rstd = 1.f / sqrtf(sq[0] * inv + p.eps);
            row_of.each([&](int i) { v[i] *= rstd * w[i]; });
            if (p.pre_b) {
                row_of.load(w, pre_b);
                row_of.each([&](int i) { v[i] += w[i]; });
            }
            row_of.store(v, p.n + at, false);
        }
        if (RING && refill) {  // no norm, no barrier yet
            __syncthreads();
            refilled();
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

// Backward of rows that a block (or a cluster of blocks, each with a slab of the columns) holds, eight values a thread.
//
// The arrays of a row are brought to shared memory some rows ahead (RING: one bulk copy an array; else plain loads of the row
// itself), and a thread keeps its columns' sums over the block's rows in registers.  A row costs two or three rounds of sums,
// about 300 clocks each, beside the 2000 that HBM takes for a row of 2048 values on every SM, so one block's rounds hide
// behind its own copies.
constexpr int kValues = 8;

// What a kernel adds up: without biases a row takes fewer instructions and registers.
enum Sums { RMS, RMS_BIAS, LAYER_BIAS };

template <Sums MODE, bool RING, bool CLUSTER>
__global__ void __launch_bounds__(kMostThreads) norm_bwd_kernel(const __grid_constant__ Backward p, const __grid_constant__ Slab slab) {
    constexpr bool VEC = RING, LAYER = MODE == LAYER_BIAS, BIAS = MODE != RMS;
    constexpr int N = kValues;
    extern __shared__ __align__(128) float ring_data[];
    __shared__ Places places;
    __shared__ float shared_sums[2][4];  // CLUSTER: this block's sums of a round
    __shared__ uint64_t full[kMostStages];
    const unsigned rank = CLUSTER ? cluster_ctarank() : 0;
    const unsigned blocks_a_row = CLUSTER ? unsigned(p.cols + slab.width - 1) / unsigned(slab.width) : 1;
    const int c0 = int(rank) * slab.width, width = min(slab.width, p.cols - c0);
    Ring ring;
    launch_next();
    if (RING) ring.init(ring_data, full, slab);
    clear_places(places);
    __syncthreads();
    launch_wait();

    const Row<N, VEC> row_of(threadIdx.x, blockDim.x, width);
    const float inv = 1.f / float(p.cols);
    const unsigned block = blockIdx.x / blocks_a_row, blocks = gridDim.x / blocks_a_row;
    const unsigned long long length = p.rows / p.groups;
    unsigned long long begin, end;
    rows_of_block(p, block, blocks, &begin, &end);
    const bool gate_each = p.gate && p.rows_per_gate == 1;
    const bool gate_bias = BIAS && p.post_b && p.gate;
    const float *post_w = p.post_w + c0, *pre_w = p.pre_w + c0, *post_b = p.post_b + c0;
    if (RING) {
        float *keep_at = ring_data + size_t(slab.stages) * slab.arrays * slab.width;
        post_w = keep_weights<VEC>(p.post_w ? post_w : nullptr, keep_at, width);
        pre_w = keep_weights<VEC>(p.dn ? pre_w : nullptr, keep_at, width);
        post_b = keep_weights<VEC>(gate_bias ? post_b : nullptr, keep_at, width);
        __syncthreads();
    }
    auto fetch = [&](int stage, unsigned long long row) {
        ring.fetch(stage, {p.r, p.h, p.dn, p.dr, gate_each ? p.gate : nullptr}, row * size_t(p.cols) + c0, width);
    };
    if (RING && threadIdx.x == 0)
        for (int i = 0; i < slab.stages && begin + i < end; ++i) fetch(i, begin + i);

    int turn = 0;
    auto round = [&](auto &v) {  // sums over the row
        constexpr int K = sizeof(v) / sizeof(v[0]);
        Rounds<false> r = {places, turn};
        r.sums(v);
        if (CLUSTER) {
            if (threadIdx.x == 0)
#pragma unroll
                for (int k = 0; k < K; ++k) shared_sums[turn][k] = v[k];
            cluster_sync_all();
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float sum = 0.f;
                for (unsigned q = 0; q < blocks_a_row; ++q) sum += ld_shared_of_rank(&shared_sums[turn][k], q);
                v[k] = sum;
            }
        }
        turn ^= 1;
    };

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
        const float *from = RING ? ring.next(p.status) : nullptr;
        row_of.load(r, RING ? from : p.r + at);
        if (p.h) row_of.load(h, RING ? from += slab.width : p.h + at);
        if (p.dn) row_of.load(dn, RING ? from += slab.width : p.dn + at);
        if (p.dr) row_of.load(dr, RING ? from += slab.width : p.dr + at);
        if (gate_each) {
            row_of.load(gate, RING ? from += slab.width : p.gate + at);
        } else if (p.gate) {
            if (gate_left == 0) {
                gate_left = p.rows_per_gate;
                gate_at += p.cols;
                row_of.load(gate, p.gate + gate_at);
            }
            --gate_left;
        }
        if (RING) fence_proxy_async_smem();  // in front of the copies behind the first round's barrier
        if (LAYER) {
            float m[2] = {0.f, 0.f};
            row_of.each([&](int i) { m[0] += r[i]; });
            if (p.post_w) row_of.each([&](int i) { m[1] += h[i]; });
            round(m);
            row_of.center(r, m[0] * inv);
            if (p.post_w) row_of.center(h, m[1] * inv);
        }
        float a[N], v[4] = {0.f, 0.f, 0.f, 0.f};  // squares of r and h, a (r - m) and a
        if (p.dn) {
            row_of.load(w, pre_w);
            row_of.each([&](int i) {
                a[i] = dn[i] * w[i];
                v[0] += r[i] * r[i];
                v[2] += a[i] * r[i];
                if (LAYER) v[3] += a[i];
            });
        }
        if (p.post_w) row_of.each([&](int i) { v[1] += h[i] * h[i]; });
        round(v);
        if (RING) {
            if (threadIdx.x == 0 && row + slab.stages < end) fetch(ring.stage, row + slab.stages);
            ring.advance();
        }
        if (!p.dr) row_of.each([&](int i) { dr[i] = 0.f; });
        if (p.dn) {
            const float rs = 1.f / sqrtf(v[0] * inv + p.eps), c_hat = v[2] * rs * inv, c_one = LAYER ? v[3] * inv : 0.f;
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
        const float hs = 1.f / sqrtf(v[1] * inv + p.eps);
        // gate times gradient; dr turns into the gate's gradient
        row_of.each([&](int i) {
            dr[i] *= p.scale;
            b[i] = p.gate ? gate[i] * dr[i] : dr[i];
        });
        if (p.post_w) {
            row_of.load(w, post_w);
            row_of.each([&](int i) {
                h[i] *= hs;
                sum_post_w[i] += b[i] * h[i];
                if (BIAS) sum_post_b[i] += b[i];
                b[i] *= w[i];
                q[0] += b[i] * h[i];
                if constexpr (LAYER) q[1] += b[i];
            });
            if (p.gate) {
                if (gate_bias) {
                    float bias[N];
                    row_of.load(bias, post_b);
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
            round(q);
            const float q_hat = q[0] * inv;
            float q_one = 0.f;
            if constexpr (LAYER) q_one = q[1] * inv;
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
    if (CLUSTER) cluster_sync_all();  // no block leaves while another may read its sums
}

// ---- rows of any length: every round of sums reads its row again (from L2, mostly) ---------------------------------
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
                block_sums<1, kThreads>(hm, sh[0]);
                hm[0] *= inv;
            }
            for (int j = threadIdx.x; j < p.cols; j += kThreads) hs[0] += (h[j] - hm[0]) * (h[j] - hm[0]);
            block_sums<1, kThreads>(hs, sh[1]);
            hs[0] = 1.f / sqrtf(hs[0] * inv + p.eps);
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
                block_sums<1, kThreads>(rm, sh[2]);
                rm[0] *= inv;
                for (int j = threadIdx.x; j < p.cols; j += kThreads) rs[0] += (r[j] - rm[0]) * (r[j] - rm[0]);
            }
            block_sums<1, kThreads>(rs, sh[3]);
            rs[0] = 1.f / sqrtf(rs[0] * inv + p.eps);
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
            block_sums<2, kThreads>(m, sh);
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
        block_sums<4, kThreads>(v, sh4);
        const float rs = 1.f / sqrtf(v[0] * inv + p.eps), hs = 1.f / sqrtf(v[1] * inv + p.eps);
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
            block_sums<2, kThreads>(q, sh2);
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

constexpr int kFoldThreads = 1024;  // 32 columns by 32 parts at a time: one round of loads for 300 blocks' sums

__global__ void __launch_bounds__(kFoldThreads) norm_fold_kernel(const __grid_constant__ Folds p) {
    __shared__ float sh[32][33];
    launch_next();
    launch_wait();
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
    const unsigned tiles = unsigned(p.cols + 31) / 32;
    unsigned long long item = blockIdx.x;
    for (int k = 0; k < p.folds; ++k) {
        const Fold &f = p.f[k];
        for (; item < f.results * tiles; item += gridDim.x) {
            const unsigned long long result = item / tiles;
            const int col = int(item - result * tiles) * 32 + lane;
            const float *src = f.partial + result * f.parts * p.cols;
            float s = 0.f;
            if (col < p.cols)
#pragma unroll 10
                for (int q = part; q < f.parts; q += 32) s += __ldcg(src + size_t(q) * p.cols + col);
            sh[part][lane] = s;
            __syncthreads();
            // warp `part` adds up column `part` of the tile
            float t = sh[lane][part];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
            const int mine = int(item - result * tiles) * 32 + part;
            if (lane == 0 && mine < p.cols) {
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

// Whether rows are whole 16-byte pieces at 16-byte addresses.
bool pieces(int cols, std::initializer_list<const void *> pointers) {
    uintptr_t at = uintptr_t(cols) * sizeof(float);
    for (const void *q : pointers) at |= reinterpret_cast<uintptr_t>(q);
    return (at & 15u) == 0;
}

template <bool LAYER>
int32_t start_forward_of(katsu_cuda_ctx *ctx, const Forward &p, bool wide, bool vec, Rows rows, const Slab &slab, size_t smem,
                         unsigned grid, unsigned block) {
    auto kernel = wide               ? norm_fwd_kernel<32, true, OF_BLOCK, LAYER>
                  : rows == BY_RING  ? norm_fwd_kernel<16, true, BY_RING, LAYER>
                  : rows == OF_BLOCK ? (vec ? norm_fwd_kernel<16, true, OF_BLOCK, LAYER> : norm_fwd_kernel<16, false, OF_BLOCK, LAYER>)
                                     : (vec ? norm_fwd_kernel<16, true, OF_WARP, LAYER> : norm_fwd_kernel<16, false, OF_WARP, LAYER>);
    if (smem) KATSU_TRY(katsu_prepare_kernel(ctx, (const void *)kernel, smem));
    return katsu_launch_chained(ctx, kernel, grid, block, smem, 1, p, slab);
}

template <bool LAYER>
int32_t start_forward(katsu_cuda_ctx *ctx, const Forward &p) {
    const bool vec = pieces(p.cols, {p.x, p.h, p.gate, p.post_w, p.post_b, p.pre_w, p.pre_b, p.r, p.n});
    const unsigned long long sms = ctx->num_sms;
    if (p.cols > kMostThreads * (vec ? 32 : 16))
        return start(ctx, norm_fwd_long_kernel<LAYER>, unsigned(p.rows < sms * 4 ? p.rows : sms * 4), kThreads, p);
    // 16 values a thread, 32 where that would take more than 512 threads; up to 512 values are one warp's
    const bool wide = p.cols > kMostThreads * 16;
    Rows rows = p.cols <= 512 ? OF_WARP : OF_BLOCK;
    const unsigned threads = rows == OF_WARP ? 128 : unsigned(katsu_div_up(katsu_div_up(p.cols, wide ? 32 : 16), 32)) * 32;
    const unsigned long long need = rows == OF_WARP ? katsu_div_up(p.rows, 4) : p.rows;
    unsigned resident = 512 / threads;  // registers: 512 threads to an SM
    if (resident > 8) resident = 8;
    const unsigned long long most = sms * resident;
    Slab slab = {};
    size_t smem = 0;
    // A block that takes several rows brings them ahead; a single one arrives sooner by plain loads (one row of 4096: 5.6 us).
    if (vec && rows == OF_BLOCK && !wide && p.rows > sms * resident) {
        slab.width = p.cols;
        slab.arrays = 1 + (p.h != nullptr) + (p.gate && p.rows_per_gate == 1);
        const size_t row = size_t(slab.arrays) * p.cols * sizeof(float);
        const size_t kept = size_t((p.post_w != nullptr) + (p.post_b != nullptr) + (p.pre_w != nullptr) + (p.pre_b != nullptr)) * p.cols * sizeof(float);
        const size_t room = kRoom / resident - 2048 > kept ? kRoom / resident - 2048 - kept : 0;
        const size_t stages = room / row < kMostStages ? room / row : kMostStages;
        if (stages >= 2) {
            rows = BY_RING;
            slab.stages = int(stages);
            smem = slab.stages * row + kept;
        }
    }
    const unsigned grid = unsigned(need < most ? need : most);
    return start_forward_of<LAYER>(ctx, p, wide, vec, rows, slab, smem, grid, threads);
}

// Which kernel a backward pass takes, and how many blocks (or clusters) go round at once.
struct BackwardShape {
    Slab slab;  // arrays 0: no ring; width 0: the kernel for rows of any length
    unsigned threads, cluster;
    size_t smem, most_blocks;
};

BackwardShape backward_shape(const katsu_cuda_ctx *ctx, const Backward &p, std::initializer_list<const void *> pointers) {
    BackwardShape s = {};
    const int most = kMostThreads * kValues;  // columns to a block
    const bool vec = pieces(p.cols, pointers);
    if (p.cols > (vec ? 4 : 1) * most) {
        s.most_blocks = size_t(ctx->num_sms) * 4;
        return s;
    }
    s.cluster = p.cols > 2 * most ? 4 : p.cols > most ? 2 : 1;
    s.slab.width = int(katsu_div_up(katsu_div_up(p.cols, s.cluster), 4)) * 4;
    s.threads = unsigned(katsu_div_up(katsu_div_up(s.slab.width, kValues), 32)) * 32;
    unsigned resident = 512 / s.threads;  // registers: 512 threads to an SM
    if (resident > 8) resident = 8;
    if (vec) {
        s.slab.arrays = 1 + (p.h != nullptr) + (p.dn != nullptr) + (p.dr != nullptr) + (p.gate && p.rows_per_gate == 1);
        const size_t row = size_t(s.slab.arrays) * s.slab.width * sizeof(float);
        const size_t kept = size_t((p.post_w != nullptr) + (p.dn != nullptr) + (p.post_b && p.gate)) * s.slab.width * sizeof(float);
        const size_t room = kRoom / resident - 2048 - kept;
        s.slab.stages = int(room / row < kMostStages ? room / row : kMostStages);
        s.smem = s.slab.stages * row + kept;
    }
    s.most_blocks = size_t(ctx->num_sms) * resident / s.cluster;
    return s;
}

template <Sums MODE>
int32_t start_backward_of(katsu_cuda_ctx *ctx, const Backward &p, const BackwardShape &s, size_t blocks) {
    auto kernel = s.cluster > 1 ? norm_bwd_kernel<MODE, true, true>
                  : s.slab.arrays ? norm_bwd_kernel<MODE, true, false> : norm_bwd_kernel<MODE, false, false>;
    if (s.smem) KATSU_TRY(katsu_prepare_kernel(ctx, (const void *)kernel, s.smem));
    return katsu_launch_chained(ctx, kernel, (unsigned)blocks * s.cluster, s.threads, s.smem, s.cluster, p, s.slab);
}

template <bool LAYER>
int32_t start_backward(katsu_cuda_ctx *ctx, const Backward &p, const BackwardShape &s, size_t blocks) {
    if (s.slab.width == 0) return start(ctx, norm_bwd_long_kernel<LAYER>, (unsigned)blocks, kThreads, p);
    const bool bias = p.post_b || p.partial[DPRE_B] || p.partial[DPOST_B];
    return LAYER ? start_backward_of<LAYER_BIAS>(ctx, p, s, blocks)
                 : bias ? start_backward_of<RMS_BIAS>(ctx, p, s, blocks) : start_backward_of<RMS>(ctx, p, s, blocks);
}

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
    for (const float *in : {x, h, gate, post_w, post_b, pre_w, pre_b})
        KATSU_REQUIRE(in == nullptr || (in != r && in != n), "an output is an input too");
    KATSU_REQUIRE(r != n, "r and n are the same buffer");
    KATSU_TRY(katsu_bind(ctx));
    Forward p = {x, h, gate, post_w, post_b, pre_w, pre_b, r, n, scale, eps, rows, gate ? rows / gate_rows : 1, (int)cols, ctx->status};
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
    float *const outs[] = {dx, dh, dgate, dpost_w, dpost_b, dpre_w, dpre_b};
    for (size_t i = 0; i < 7; ++i) {
        if (outs[i] == nullptr) continue;
        for (size_t j = 0; j < i; ++j) KATSU_REQUIRE(outs[i] != outs[j], "two outputs are the same buffer");
        for (const float *in : {r, h, gate, post_w, post_b, pre_w, dr, dn})
            KATSU_REQUIRE(in != outs[i], "an output is an input too");
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
    p.add_dx = accumulate & KATSU_BLOCK_DX; p.add_dh = accumulate & KATSU_BLOCK_DH; p.add_dgate = adds[DGATE];
    p.gate_of_row = dgate && gate_rows == rows;
    p.groups = dgate && !p.gate_of_row ? gate_rows : 1;
    p.status = ctx->status;
    const BackwardShape shape = backward_shape(ctx, p, {r, h, gate, post_w, post_b, pre_w, dr, dn, dx, dh, dgate});
    const size_t want = shape.most_blocks < rows ? shape.most_blocks : rows;
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
    KATSU_TRY(kind == KATSU_NORM_LAYER ? start_backward<true>(ctx, p, shape, blocks) : start_backward<false>(ctx, p, shape, blocks));
    if (folds.folds == 0) return KATSU_OK;
    unsigned long long items = 0;
    for (int k = 0; k < folds.folds; ++k) items += folds.f[k].results * katsu_div_up(cols, 32);
    const unsigned long long most = (unsigned long long)ctx->num_sms * 2;
    return start(ctx, norm_fold_kernel, unsigned(items < most ? items : most), kFoldThreads, folds);
}
