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
// N values of a row for each of T threads: pieces of four, T pieces apart (VEC: 16-byte accesses, the row's pieces are whole), or
// single values T apart.  `width` values from `at` on; what lies behind them is 0 and not stored.
template <int N, bool VEC>
__device__ __forceinline__ void load_row(float (&v)[N], const float *at, int t, int T, int width) {
#pragma unroll
    for (int i = 0; i < N; i += VEC ? 4 : 1) {
        if (VEC) {
            const int j = 4 * (t + i / 4 * T);
            const float4 f = j < width ? *reinterpret_cast<const float4 *>(at + j) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
        } else {
            const int j = t + i * T;
            v[i] = j < width ? at[j] : 0.f;
        }
    }
}

template <int N, bool VEC>
__device__ __forceinline__ void store_row(const float (&v)[N], float *at, int t, int T, int width, bool add) {
#pragma unroll
    for (int i = 0; i < N; i += VEC ? 4 : 1) {
        if (VEC) {
            const int j = 4 * (t + i / 4 * T);
            if (j >= width) break;
            float4 f = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            if (add) {
                const float4 old = *reinterpret_cast<const float4 *>(at + j);
                f.x += old.x; f.y += old.y; f.z += old.z; f.w += old.w;
            }
            *reinterpret_cast<float4 *>(at + j) = f;
        } else {
            const int j = t + i * T;
            if (j >= width) break;
            at[j] = add ? at[j] + v[i] : v[i];
        }
    }
}

// Whether value i of this thread is one of the row's.
template <bool VEC>
__device__ __forceinline__ bool in_row(int i, int t, int T, int width) {
    return (VEC ? 4 * (t + i / 4 * T) : t + i * T) < width;
}

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

template <int N, bool VEC, bool WARP, bool LAYER>
__global__ void __launch_bounds__(kMostThreads) norm_fwd_kernel(const __grid_constant__ Forward p) {
    __shared__ Places places;
    launch_next();
    if (!WARP) {
        clear_places(places);
        __syncthreads();
    }
    launch_wait();
    Rounds<WARP> rounds = {places, 0};
    const int T = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const unsigned per_block = WARP ? blockDim.x >> 5 : 1;
    const float inv = 1.f / float(p.cols);
    for (unsigned long long row = (unsigned long long)blockIdx.x * per_block + (WARP ? threadIdx.x >> 5 : 0); row < p.rows;
         row += (unsigned long long)gridDim.x * per_block) {
        const size_t at = row * size_t(p.cols);
        float v[N], u[N], w[N];
        load_row<N, VEC>(v, p.x + at, t, T, p.cols);
        if (p.h) {
            load_row<N, VEC>(u, p.h + at, t, T, p.cols);
            float g[N];
            if (p.gate) load_row<N, VEC>(g, p.gate + row / p.rows_per_gate * p.cols, t, T, p.cols);
            if (p.post_w) {
                float m[1] = {0.f}, sq[1] = {0.f};
                if (LAYER) {
#pragma unroll
                    for (int i = 0; i < N; ++i) m[0] += u[i];
                    rounds.sums(m);
                    m[0] *= inv;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (LAYER) u[i] = in_row<VEC>(i, t, T, p.cols) ? u[i] - m[0] : 0.f;
                    sq[0] += u[i] * u[i];
                }
                load_row<N, VEC>(w, p.post_w, t, T, p.cols);
                rounds.sums(sq);
                const float rstd = 1.f / sqrtf(sq[0] * inv + p.eps);
#pragma unroll
                for (int i = 0; i < N; ++i) u[i] *= rstd * w[i];
                if (p.post_b) {
                    load_row<N, VEC>(w, p.post_b, t, T, p.cols);
#pragma unroll
                    for (int i = 0; i < N; ++i) u[i] += w[i];
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += p.scale * (p.gate ? g[i] * u[i] : u[i]);
            store_row<N, VEC>(v, p.r + at, t, T, p.cols, false);
        }
        if (!p.n) continue;
        float m[1] = {0.f}, sq[1] = {0.f};
        if (LAYER) {
#pragma unroll
            for (int i = 0; i < N; ++i) m[0] += v[i];
            rounds.sums(m);
            m[0] *= inv;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (LAYER) v[i] = in_row<VEC>(i, t, T, p.cols) ? v[i] - m[0] : 0.f;
            sq[0] += v[i] * v[i];
        }
        load_row<N, VEC>(w, p.pre_w, t, T, p.cols);
        rounds.sums(sq);
        const float rstd = 1.f / sqrtf(sq[0] * inv + p.eps);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= rstd * w[i];
        if (p.pre_b) {
            load_row<N, VEC>(w, p.pre_b, t, T, p.cols);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += w[i];
        }
        store_row<N, VEC>(v, p.n + at, t, T, p.cols, false);
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

struct Slab {
    int width, arrays, stages;  // columns to a block; arrays of the ring and its depth in rows
};

template <Sums MODE, bool RING, bool CLUSTER>
__global__ void __launch_bounds__(kMostThreads) norm_bwd_kernel(const __grid_constant__ Backward p, const __grid_constant__ Slab slab) {
    constexpr bool VEC = RING, LAYER = MODE == LAYER_BIAS, BIAS = MODE != RMS;
    constexpr int N = kValues;
    extern __shared__ __align__(128) float ring[];
    __shared__ Places places;
    __shared__ float shared_sums[2][4];  // CLUSTER: this block's sums of a round
    __shared__ uint64_t full[8];
    const int T = blockDim.x, t = threadIdx.x;
    const unsigned rank = CLUSTER ? cluster_ctarank() : 0, blocks_a_row = CLUSTER ? unsigned(p.cols + slab.width - 1) / unsigned(slab.width) : 1;
    const int c0 = int(rank) * slab.width, width = min(slab.width, p.cols - c0);
    launch_next();
    if (RING && t == 0) {
        for (int s = 0; s < slab.stages; ++s) mbar_init(&full[s], 1);
        mbar_init_fence();
    }
    clear_places(places);
    __syncthreads();
    launch_wait();

    const float inv = 1.f / float(p.cols);
    const unsigned block = blockIdx.x / blocks_a_row, blocks = gridDim.x / blocks_a_row;
    const unsigned long long length = p.rows / p.groups;
    unsigned long long begin, end;
    rows_of_block(p, block, blocks, &begin, &end);
    const bool gate_each = p.gate && p.rows_per_gate == 1;
    // arrays in the ring: r, then those of h, dn, dr and a gate for each row that there are
    auto fetch = [&](unsigned long long row) {
        const int s = int((row - begin) % slab.stages);
        const uint32_t bytes = uint32_t(width) * 4;
        float *to = ring + size_t(s) * slab.arrays * slab.width;
        const size_t at = row * size_t(p.cols) + c0;
        mbar_arrive_expect_tx(&full[s], bytes * slab.arrays);
        for (const float *src : {p.r, p.h, p.dn, p.dr, gate_each ? p.gate : nullptr})
            if (src) {
                bulk_load(to, src + at, bytes, &full[s]);
                to += slab.width;
            }
    };
    if (RING && t == 0)
        for (unsigned long long row = begin; row < end && row < begin + slab.stages; ++row) fetch(row);

    int turn = 0;
    auto round = [&](auto &v) {  // sums over the row
        constexpr int K = sizeof(v) / sizeof(v[0]);
        Rounds<false> r = {places, turn};
        r.sums(v);
        if (CLUSTER) {
            if (t == 0)
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

    float gate[N] = {}, sum_gate[N] = {}, sum_pre_w[N] = {}, sum_pre_b[N] = {}, sum_post_w[N] = {}, sum_post_b[N] = {};
    for (unsigned long long row = begin; row < end; ++row) {
        const size_t at = row * size_t(p.cols) + c0;
        float r[N], h[N], dn[N] = {}, dr[N] = {}, w[N];
        if (RING) {
            const unsigned long long i = row - begin;
            const int s = int(i % slab.stages);
            // (a wait that gives up leaves wrong values behind, which the next synchronising call reports)
            mbar_wait_warp(&full[s], uint32_t(i / slab.stages) & 1u, p.status, 191);
            const float *from = ring + size_t(s) * slab.arrays * slab.width;
            load_row<N, VEC>(r, from, t, T, width);
            if (p.h) load_row<N, VEC>(h, from += slab.width, t, T, width);
            if (p.dn) load_row<N, VEC>(dn, from += slab.width, t, T, width);
            if (p.dr) load_row<N, VEC>(dr, from += slab.width, t, T, width);
            if (gate_each) load_row<N, VEC>(gate, from += slab.width, t, T, width);
            fence_proxy_async_smem();  // in front of the copies behind the first round's barrier
        } else {
            load_row<N, VEC>(r, p.r + at, t, T, width);
            if (p.h) load_row<N, VEC>(h, p.h + at, t, T, width);
            if (p.dn) load_row<N, VEC>(dn, p.dn + at, t, T, width);
            if (p.dr) load_row<N, VEC>(dr, p.dr + at, t, T, width);
            if (gate_each) load_row<N, VEC>(gate, p.gate + at, t, T, width);
        }
        if (p.gate && !gate_each && (row == begin || row % p.rows_per_gate == 0))
            load_row<N, VEC>(gate, p.gate + row / p.rows_per_gate * p.cols + c0, t, T, width);
        if (!p.h)
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = 0.f;
        if (LAYER) {
            float m[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < N; ++i) {
                m[0] += r[i];
                m[1] += h[i];
            }
            round(m);
            const float mr = m[0] * inv, mh = p.post_w ? m[1] * inv : 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool in = in_row<VEC>(i, t, T, width);
                r[i] = in ? r[i] - mr : 0.f;
                h[i] = in ? h[i] - mh : 0.f;
            }
        }
        float a[N], v[4] = {0.f, 0.f, 0.f, 0.f};  // squares of r and h, a (r - m) and a
        if (p.dn) load_row<N, VEC>(w, p.pre_w + c0, t, T, width);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            a[i] = p.dn ? dn[i] * w[i] : 0.f;
            v[0] += r[i] * r[i];
            v[1] += h[i] * h[i];
            v[2] += a[i] * r[i];
            if (LAYER) v[3] += a[i];
        }
        round(v);
        if (RING && t == 0 && row + slab.stages < end) fetch(row + slab.stages);
        const float rs = 1.f / sqrtf(v[0] * inv + p.eps), hs = 1.f / sqrtf(v[1] * inv + p.eps);
        const float c_hat = v[2] * rs * inv, c_one = LAYER ? v[3] * inv : 0.f;
        if (p.dn)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float hat = r[i] * rs;
                dr[i] += rs * (a[i] - hat * c_hat - c_one);  // all of r's gradient from here on
                sum_pre_w[i] += dn[i] * hat;
                if (BIAS) sum_pre_b[i] += dn[i];
            }
        if (p.dx) store_row<N, VEC>(dr, p.dx + at, t, T, width, p.add_dx);
        if (!p.h) continue;
        float q[LAYER ? 2 : 1] = {}, b[N];  // b h^ and b behind the block
        if (p.post_w) {
            load_row<N, VEC>(w, p.post_w + c0, t, T, width);
            float bias[N] = {};
            if (BIAS && p.post_b && (p.dgate || p.partial[DGATE])) load_row<N, VEC>(bias, p.post_b + c0, t, T, width);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float sd = p.scale * dr[i], du = p.gate ? gate[i] * sd : sd;
                h[i] *= hs;
                b[i] = in_row<VEC>(i, t, T, width) ? du * w[i] : 0.f;
                q[0] += b[i] * h[i];
                if constexpr (LAYER) q[1] += b[i];
                sum_post_w[i] += du * h[i];
                if (BIAS) sum_post_b[i] += du;
                dr[i] = sd * (h[i] * w[i] + bias[i]);  // the gate's
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float sd = p.scale * dr[i], u = h[i];
                b[i] = p.gate ? gate[i] * sd : sd;
                dr[i] = sd * u;
            }
        }
        if (p.gate_of_row) {
            store_row<N, VEC>(dr, p.dgate + at, t, T, width, p.add_dgate);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) sum_gate[i] += dr[i];
            if (p.dgate && (row + 1) % length == 0) {
                store_row<N, VEC>(sum_gate, p.dgate + row / length * p.cols + c0, t, T, width, p.add_dgate);
#pragma unroll
                for (int i = 0; i < N; ++i) sum_gate[i] = 0.f;
            }
        }
        if (!p.dh) continue;
        if (p.post_w) {
            round(q);
            float q_one = 0.f;
            if constexpr (LAYER) q_one = q[1] * inv;
            const float q_hat = q[0] * inv;
#pragma unroll
            for (int i = 0; i < N; ++i) b[i] = hs * (b[i] - h[i] * q_hat - q_one);
        }
        store_row<N, VEC>(b, p.dh + at, t, T, width, p.add_dh);
    }
    const size_t mine = size_t(block) * p.cols + c0;
    if (p.partial[DPRE_W]) store_row<N, VEC>(sum_pre_w, p.partial[DPRE_W] + mine, t, T, width, false);
    if (BIAS && p.partial[DPRE_B]) store_row<N, VEC>(sum_pre_b, p.partial[DPRE_B] + mine, t, T, width, false);
    if (p.partial[DPOST_W]) store_row<N, VEC>(sum_post_w, p.partial[DPOST_W] + mine, t, T, width, false);
    if (BIAS && p.partial[DPOST_B]) store_row<N, VEC>(sum_post_b, p.partial[DPOST_B] + mine, t, T, width, false);
    if (p.partial[DGATE]) store_row<N, VEC>(sum_gate, p.partial[DGATE] + mine, t, T, width, false);
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
    KATSU_TRY(katsu_prepare_kernel(ctx, (const void *)kernel, 0));
    return katsu_launch_chained(ctx, kernel, grid, block, 0, 1, args...);
}

// Whether rows are whole 16-byte pieces at 16-byte addresses.
bool pieces(int cols, std::initializer_list<const void *> pointers) {
    uintptr_t at = uintptr_t(cols) * sizeof(float);
    for (const void *q : pointers) at |= reinterpret_cast<uintptr_t>(q);
    return (at & 15u) == 0;
}

template <int N, bool LAYER>
int32_t start_forward_of(katsu_cuda_ctx *ctx, const Forward &p, bool vec, bool warp, unsigned grid, unsigned block) {
    if (warp) return start(ctx, vec ? norm_fwd_kernel<16, true, true, LAYER> : norm_fwd_kernel<16, false, true, LAYER>, grid, block, p);
    return start(ctx, vec ? norm_fwd_kernel<N, true, false, LAYER> : norm_fwd_kernel<N, false, false, LAYER>, grid, block, p);
}

template <bool LAYER>
int32_t start_forward(katsu_cuda_ctx *ctx, const Forward &p) {
    const bool vec = pieces(p.cols, {p.x, p.h, p.gate, p.post_w, p.post_b, p.pre_w, p.pre_b, p.r, p.n});
    const unsigned long long sms = ctx->num_sms;
    if (p.cols > kMostThreads * 32)
        return start(ctx, norm_fwd_long_kernel<LAYER>, unsigned(p.rows < sms * 8 ? p.rows : sms * 8), kThreads, p);
    // 16 values a thread, 32 where that would take more than 512 threads; up to 512 values are one warp's
    const bool warp = p.cols <= 512, wide = p.cols > kMostThreads * 16;
    const unsigned threads = warp ? 128 : unsigned(katsu_div_up(katsu_div_up(p.cols, wide ? 32 : 16), 32)) * 32;
    const unsigned long long need = warp ? katsu_div_up(p.rows, 4) : p.rows, most = sms * (2048 / threads);
    const unsigned grid = unsigned(need < most ? need : most);
    return wide ? start_forward_of<32, LAYER>(ctx, p, vec, warp, grid, threads) : start_forward_of<16, LAYER>(ctx, p, vec, warp, grid, threads);
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
        const size_t row = size_t(s.slab.arrays) * s.slab.width * sizeof(float), room = size_t(216) * 1024 / resident - 1024;
        s.slab.stages = int(room / row < 4 ? room / row : 4);
        s.smem = s.slab.stages * row;
    }
    s.most_blocks = size_t(ctx->num_sms) * resident / s.cluster;
    return s;
}

template <Sums MODE>
int32_t start_backward_of(katsu_cuda_ctx *ctx, const Backward &p, const BackwardShape &s, size_t blocks) {
    auto kernel = s.cluster > 1 ? norm_bwd_kernel<MODE, true, true>
                  : s.slab.arrays ? norm_bwd_kernel<MODE, true, false> : norm_bwd_kernel<MODE, false, false>;
    KATSU_TRY(katsu_prepare_kernel(ctx, (const void *)kernel, s.smem));
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
    Forward p = {x, h, gate, post_w, post_b, pre_w, pre_b, r, n, scale, eps, rows, gate ? rows / gate_rows : 1, (int)cols};
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
