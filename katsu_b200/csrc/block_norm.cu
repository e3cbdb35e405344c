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

#include "common.cuh"
#include "launch.cuh"

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

// First and last row of the block's share; a block has one piece of a group or several whole groups.
__device__ __forceinline__ void rows_of_block(const Backward &p, unsigned long long *begin, unsigned long long *end) {
    const unsigned long long length = p.rows / p.groups;
    if (p.slices > 1) {
        const unsigned long long group = blockIdx.x / p.slices, s = blockIdx.x % p.slices;
        *begin = group * length + length * s / p.slices;
        *end = group * length + length * (s + 1) / p.slices;
    } else {
        *begin = p.groups * blockIdx.x / gridDim.x * length;
        *end = p.groups * (blockIdx.x + 1) / gridDim.x * length;
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
    rows_of_block(p, &begin, &end);
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

__global__ void __launch_bounds__(kThreads) norm_fold_kernel(const __grid_constant__ Folds p) {
    __shared__ float sh[8][33];
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
#pragma unroll 8
                for (int q = part; q < f.parts; q += 8) s += __ldcg(src + size_t(q) * p.cols + col);
            sh[part][lane] = s;
            __syncthreads();
            if (part == 0 && col < p.cols) {
                float t = 0.f;
#pragma unroll
                for (int q = 0; q < 8; ++q) t += sh[q][lane];
                float *o = f.out + result * p.cols + col;
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
    const size_t most = size_t(ctx->num_sms) * 8;
    const unsigned blocks = unsigned(rows < most ? rows : most);
    auto kernel = kind == KATSU_NORM_LAYER ? norm_fwd_long_kernel<true> : norm_fwd_long_kernel<false>;
    return start(ctx, kernel, blocks, kThreads, p);
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
    // one block a row at first, then more rows to a block: a block's sums over rows are written and read once more
    const size_t want = size_t(ctx->num_sms) * 4 < rows ? size_t(ctx->num_sms) * 4 : rows;
    size_t blocks;
    if (p.gate_of_row || dgate == nullptr || p.groups < want) {
        p.slices = (int)katsu_div_up(want, p.groups);
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
    auto kernel = kind == KATSU_NORM_LAYER ? norm_bwd_long_kernel<true> : norm_bwd_long_kernel<false>;
    KATSU_TRY(start(ctx, kernel, (unsigned)blocks, kThreads, p));
    if (folds.folds == 0) return KATSU_OK;
    unsigned long long items = 0;
    for (int k = 0; k < folds.folds; ++k) items += folds.f[k].results * katsu_div_up(cols, 32);
    const unsigned long long most = (unsigned long long)ctx->num_sms * 8;
    return start(ctx, norm_fold_kernel, unsigned(items < most ? items : most), kThreads, folds);
}
