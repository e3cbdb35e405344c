// The norm over all gradients of a step, clipping by it, and the SGD step with clipped gradients.
//
//   norm = sqrt(sum over all tensors of g^2)      c = max_norm / norm where that is below 1      g' = c g      w -= lr (c g)
//
// Two launches (and one more pair for every 512 tensors): the first leaves a partial sum of squares a block, the blocks of the
// second fold these for themselves and then scale or step.  With more blocks than are resident at once a launch between the two
// folds once for all.  The addresses travel as a kernel parameter, so nothing on the host has to outlive the call and a captured
// call keeps them.  Bound: HBM; 240 tensors of 1.2 GB and their weights take 169 us for the squares (7.1 TB/s) and 506 for the
// step (7.2 TB/s, the gradients read again but for what L2 still has).
//
// Squares are summed in 64 bits: 1e-30 and 1e30 neither vanish nor overflow, the sum of 1e9 values keeps more bits than the
// f32 result shows, and a sum that is not finite means exactly that a gradient is not.  It costs nothing beside the loads: a
// conversion and a multiply-add a value, 16 and 64 lanes a clock and SM, where the memory brings 6 values.
#include <math.h>

#include <algorithm>
#include <vector>

#include "common.cuh"
#include "launch.cuh"

namespace {

constexpr int kThreads = 256;
constexpr unsigned kUnit = 4 * kThreads;  // values of one 16-byte access a thread
constexpr int kBatch = 4;                 // units whose loads are on their way together
constexpr int kMaxTensors = 512;          // a launch (14 KiB of parameters)
constexpr int kFewTensors = 32;           // (1 KiB: the launch of a large parameter block takes longer)

// Tensors of one launch.  Unit u of a tensor has the values whose place behind the 16-byte boundary at or in front of the
// tensor is u * kUnit .. u * kUnit + kUnit - 1, so that 16-byte accesses fit tensors at any address.
template <int N>
struct Tensors {
    const float *src[N];
    float *dst[N];
    unsigned long long count[N];
    unsigned first[N + 1];  // units in front of the tensor
    int tensors;
};

enum Apply { CLIP, STEP };

__device__ __forceinline__ double block_sum(double v, double *sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int q = 0; q < kThreads / 32; ++q) t += sh[q];
    return t;
}

// Units begin .. end - 1, of all tensors counted through, as batches of one tensor's: the first batch, and the one behind it.
struct Batch {
    int tensor, units;  // units 0: none is left
    unsigned unit;      // first one, of the tensor's
    unsigned begin, end;
};

template <int N>
__device__ __forceinline__ void next_batch(const Tensors<N> &t, Batch *b) {
    b->units = 0;
    if (b->begin >= b->end) return;
    while (b->begin >= t.first[b->tensor + 1]) ++b->tensor;
    b->unit = b->begin - t.first[b->tensor];
    b->units = int(min(min(b->end, t.first[b->tensor + 1]) - b->begin, unsigned(kBatch)));
    b->begin += b->units;
}

template <int N>
__device__ __forceinline__ Batch first_batch(const Tensors<N> &t, unsigned begin, unsigned end) {
    int lo = 0, hi = t.tensors - 1;  // the last tensor whose first unit is not behind `begin` (empty tensors are left out)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= begin) lo = mid;
        else hi = mid - 1;
    }
    Batch b = {lo, 0, 0, begin, end};
    next_batch(t, &b);
    return b;
}

__device__ __forceinline__ unsigned lead_of(const float *p) { return unsigned(reinterpret_cast<uintptr_t>(p) >> 2) & 3u; }

// partial[block] = the block's sum of squares.
template <int N>
__global__ void __launch_bounds__(kThreads) squares_kernel(const __grid_constant__ Tensors<N> t, double *partial, int waves) {
    if (!waves) launch_next();
    launch_wait();
    double acc = 0.0;
    // runs differ by one unit, so no block has a batch more to do than the others
    const unsigned long long units = t.first[t.tensors];
    for (Batch b = first_batch(t, unsigned(units * blockIdx.x / gridDim.x), unsigned(units * (blockIdx.x + 1) / gridDim.x)); b.units;
         next_batch(t, &b)) {
        const int i = b.tensor;
        const float *src = t.src[i];
        const unsigned lead = lead_of(src);
        const float *base = src - lead;
        const unsigned long long begin = (unsigned long long)b.unit * kUnit, end = lead + t.count[i];
        float4 v[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const unsigned long long a = begin + 4ull * (threadIdx.x + j * kThreads);
            v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (j >= b.units) continue;
            if (a >= lead && a + 4 <= end) {
                v[j] = __ldg(reinterpret_cast<const float4 *>(base + a));
            } else {
                if (a >= lead && a < end) v[j].x = __ldg(base + a);
                if (a + 1 >= lead && a + 1 < end) v[j].y = __ldg(base + a + 1);
                if (a + 2 >= lead && a + 2 < end) v[j].z = __ldg(base + a + 2);
                if (a + 3 >= lead && a + 3 < end) v[j].w = __ldg(base + a + 3);
            }
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            acc = fma((double)v[j].x, (double)v[j].x, acc);
            acc = fma((double)v[j].y, (double)v[j].y, acc);
            acc = fma((double)v[j].z, (double)v[j].z, acc);
            acc = fma((double)v[j].w, (double)v[j].w, acc);
        }
    }
    __shared__ double sh[kThreads / 32];
    acc = block_sum(acc, sh);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// The sum of all partials, the same in every block; the caller's threads all get it.
template <int BATCH>
__device__ __forceinline__ double fold(const double *partial, int parts) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < parts; i += BATCH * kThreads) {  // a batch is on its way together, the last one too
        double v[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) v[j] = i + j * kThreads < parts ? __ldcg(partial + i + j * kThreads) : 0.0;
#pragma unroll
        for (int j = 0; j < BATCH; ++j) acc += v[j];
    }
    __shared__ double sh[kThreads / 32];
    return block_sum(acc, sh);
}

// What gradients are multiplied by; NaN: one of them is no number.
__device__ __forceinline__ float factor_of(double sum, double norm, float max_norm) {
    if (!isfinite(sum)) return __int_as_float(0x7fffffff);
    return norm > (double)max_norm ? (float)((double)max_norm / norm) : 1.f;
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double *partial, int parts, float max_norm, float *norm, float *factor) {
    launch_next();
    launch_wait();
    const double sum = fold<16>(partial, parts), total = sqrt(sum);
    if (threadIdx.x != 0) return;
    norm[0] = (float)total;
    if (factor) *factor = factor_of(sum, total, max_norm);
}

// g and the product are rounded as katsu_cuda_clip_grads followed by katsu_cuda_sgd_step round them.
template <Apply OP>
__device__ __forceinline__ float applied(float g, float w, float c, float lr) {
    const float clipped = OP == CLIP && c == 1.f ? g : __fmul_rn(g, c);  // (a product with 1 is not all of a NaN's bits)
    return OP == CLIP ? clipped : w - __fmul_rn(lr, clipped);
}

// A block takes a batch of units (of several tensors where they are short), the last one first: what the pass over the squares
// has read last is still in L2.  The first loads are on their way before the block looks at the factor or folds the sums for it
// (looking first, the 240 tensors' step took 682 us, at 5.3 TB/s).
template <Apply OP, int N>
__global__ void __launch_bounds__(kThreads) apply_kernel(const __grid_constant__ Tensors<N> t, const double *partial, int parts,
                                                         const float *factor, float max_norm, float lr, float *norm) {
    if (factor == nullptr) launch_next();  // (else the grid goes in waves)
    launch_wait();
    const unsigned begin_unit = (gridDim.x - 1 - blockIdx.x) * kBatch;
    Batch b = first_batch(t, begin_unit, min(begin_unit + kBatch, t.first[t.tensors]));
    // One thread reads the factor: read by all, its one place in L2 had 600 000 requests to answer and held up the rest (633 us).
    __shared__ float shared_factor;
    if (factor != nullptr && threadIdx.x == 0) shared_factor = __ldcg(factor);
    float c = 0.f;
    bool known = false;
    for (; b.units; next_batch(t, &b)) {
        const float *src = t.src[b.tensor];
        float *dst = t.dst[b.tensor];
        const unsigned lead = lead_of(src);
        const unsigned long long begin = (unsigned long long)b.unit * kUnit, end = lead + t.count[b.tensor];
        const float *sb = src - lead;
        float *db = dst - lead;
        const bool whole = lead_of(dst) == lead;
        float4 g[kBatch], w[kBatch];
        if (whole)
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const unsigned long long a = begin + 4ull * (threadIdx.x + j * kThreads);
                if (j < b.units && a >= lead && a + 4 <= end) {
                    g[j] = *reinterpret_cast<const float4 *>(sb + a);
                    if (OP == STEP) w[j] = *reinterpret_cast<const float4 *>(db + a);
                }
            }
        if (!known && factor != nullptr) {
            __syncthreads();
            c = shared_factor;
        } else if (!known) {
            const double sum = fold<3>(partial, parts), total = sqrt(sum);
            if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)total;
            c = factor_of(sum, total, max_norm);
        }
        known = true;
        const bool finite = !isnan(c);
        if (OP == STEP && !finite) return;
        const float scale = finite ? c : 1.f;
        if (OP == CLIP && scale == 1.f && src == dst) continue;
        if (whole) {
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const unsigned long long a = begin + 4ull * (threadIdx.x + j * kThreads);
                if (j >= b.units) continue;
                if (a >= lead && a + 4 <= end) {
                    float4 o;
                    o.x = applied<OP>(g[j].x, OP == STEP ? w[j].x : 0.f, scale, lr);
                    o.y = applied<OP>(g[j].y, OP == STEP ? w[j].y : 0.f, scale, lr);
                    o.z = applied<OP>(g[j].z, OP == STEP ? w[j].z : 0.f, scale, lr);
                    o.w = applied<OP>(g[j].w, OP == STEP ? w[j].w : 0.f, scale, lr);
                    *reinterpret_cast<float4 *>(db + a) = o;
                } else {
                    for (unsigned long long e = a; e < a + 4; ++e)
                        if (e >= lead && e < end) db[e] = applied<OP>(sb[e], OP == STEP ? db[e] : 0.f, scale, lr);
                }
            }
        } else {
            const unsigned long long last = min(begin + (unsigned long long)b.units * kUnit, end);
            for (unsigned long long e = begin + threadIdx.x; e < last; e += kThreads)
                if (e >= lead) db[e] = applied<OP>(sb[e], OP == STEP ? db[e] : 0.f, scale, lr);
        }
    }
}

template <int N>
size_t take(Tensors<N> *t, const float *const *src, float *const *dst, const size_t *counts, size_t from, size_t tensors) {
    int k = 0;
    unsigned long long units = 0;
    size_t i = from;
    for (; i < tensors && k < N; ++i) {
        if (counts[i] == 0) continue;
        const unsigned long long lead = (reinterpret_cast<uintptr_t>(src[i]) >> 2) & 3u;
        const unsigned long long more = (lead + counts[i] + kUnit - 1) / kUnit;
        if (k > 0 && units + more > 0xf0000000ull) break;
        t->src[k] = src[i];
        t->dst[k] = dst ? dst[i] : nullptr;
        t->count[k] = counts[i];
        t->first[k] = (unsigned)units;
        units += more;
        t->first[++k] = (unsigned)units;
    }
    t->tensors = k;
    return i;
}

// Blocks with at most a batch of units each.
unsigned blocks_for(unsigned units) { return units / kBatch + (units % kBatch != 0); }

enum What { NORM_ONLY, CLIPPED, STEPPED };

template <int N>
int32_t run(katsu_cuda_ctx *ctx, What what, const float *const *grads, float *const *dst, const size_t *counts, size_t tensors,
            float lr, float max_norm, float *norm) {
    Tensors<N> t;
    // Partial sums of a launch: more blocks than go round at once, which the hardware hands out as others end, read 15 % faster
    // than each SM's share in one piece (1.2 GB: 170 us, 186), and 9 500 numbers are folded in 4 us.
    const unsigned most = unsigned(ctx->num_sms) * 64;
    size_t sums = 0, blocks = 0;
    for (size_t i = 0; i < tensors;) {
        i = take(&t, grads, dst, counts, i, tensors);
        blocks += blocks_for(t.first[t.tensors]);
        sums += std::min(blocks_for(t.first[t.tensors]), most);
    }
    float *scratch = nullptr;
    KATSU_TRY(katsu_scratch(ctx, sums * 2 + 2, &scratch));
    double *partial = reinterpret_cast<double *>(scratch + 2);
    const bool waves = blocks > size_t(ctx->num_sms) * 4;  // (blocks of the last kernel that are resident at once)
    int parts = 0;
    for (size_t i = 0; i < tensors;) {
        i = take(&t, grads, dst, counts, i, tensors);
        if (t.tensors == 0) break;
        const unsigned grid = std::min(blocks_for(t.first[t.tensors]), most);
        KATSU_TRY(katsu_launch(ctx, !waves, squares_kernel<N>, grid, kThreads, 0, 1, t, partial + parts, waves ? 1 : 0));
        parts += (int)grid;
    }
    const bool between = what != NORM_ONLY && waves;
    float *factor = between ? scratch : nullptr;
    if (what == NORM_ONLY || between || parts == 0) {
        KATSU_TRY(katsu_launch_chained(ctx, norm_kernel, 1, kThreads, 0, 1, partial, parts, max_norm, norm, factor));
    }
    if (what == NORM_ONLY) return KATSU_OK;
    auto kernel = what == CLIPPED ? apply_kernel<CLIP, N> : apply_kernel<STEP, N>;
    for (size_t i = 0; i < tensors;) {
        const bool first = i == 0;
        i = take(&t, grads, dst, counts, i, tensors);
        if (t.tensors == 0) break;
        KATSU_TRY(katsu_launch(ctx, !waves, kernel, blocks_for(t.first[t.tensors]), kThreads, 0, 1, t, partial, parts, factor,
                                       max_norm, lr, first ? norm : nullptr));
    }
    return KATSU_OK;
}

struct Range {
    uintptr_t begin, end;
    size_t tensor;
};

// Whether the written buffers are apart from each other and from what is read; written[i] may be read[i] itself.
bool apart(const float *const *read, float *const *written, const size_t *counts, size_t tensors, bool in_place) {
    std::vector<Range> w;
    w.reserve(tensors);
    for (size_t i = 0; i < tensors; ++i)
        if (counts[i]) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(written[i]);
            w.push_back({at, at + counts[i] * sizeof(float), i});
        }
    std::sort(w.begin(), w.end(), [](const Range &a, const Range &b) { return a.begin < b.begin; });
    for (size_t i = 1; i < w.size(); ++i)
        if (w[i].begin < w[i - 1].end) return false;
    for (size_t i = 0; i < tensors; ++i) {
        if (!counts[i]) continue;
        const uintptr_t at = reinterpret_cast<uintptr_t>(read[i]), end = at + counts[i] * sizeof(float);
        // the written buffers that this one meets: they are in order, and apart
        auto it = std::upper_bound(w.begin(), w.end(), at, [](uintptr_t v, const Range &r) { return v < r.end; });
        for (; it != w.end() && it->begin < end; ++it)
            if (!in_place || it->tensor != i || it->begin != at) return false;
    }
    return true;
}

int32_t checked(katsu_cuda_ctx *ctx, What what, const float *const *grads, float *const *dst, const size_t *counts,
                size_t tensors, float lr, float max_norm, float *norm) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_REQUIRE(norm != nullptr, "norm is null");
    KATSU_REQUIRE(((uintptr_t)norm & 3u) == 0, "norm is not at a whole float");
    KATSU_REQUIRE(tensors == 0 || (grads != nullptr && counts != nullptr), "null array of gradients or counts");
    KATSU_REQUIRE(tensors == 0 || what == NORM_ONLY || dst != nullptr, "null array of outputs or weights");
    KATSU_REQUIRE(what == NORM_ONLY || max_norm >= 0.f, "max_norm must be 0 or more");
    size_t live = 0;
    const auto holds_norm = [&](const float *p, size_t count) { return norm + 1 > p && norm < p + count; };
    for (size_t i = 0; i < tensors; ++i) {
        if (counts[i] == 0) continue;
        KATSU_REQUIRE(counts[i] < (size_t(1) << 41), "count out of range");
        KATSU_REQUIRE(grads[i] != nullptr, "null gradient");
        KATSU_REQUIRE(((uintptr_t)grads[i] & 3u) == 0, "a gradient is not at a whole float");
        KATSU_REQUIRE(!holds_norm(grads[i], counts[i]), "norm lies in a gradient");
        if (what != NORM_ONLY) {
            KATSU_REQUIRE(dst[i] != nullptr, "null output or weight");
            KATSU_REQUIRE(((uintptr_t)dst[i] & 3u) == 0, "an output or weight is not at a whole float");
            KATSU_REQUIRE(!holds_norm(dst[i], counts[i]), "norm lies in an output or weight");
        }
        ++live;
    }
    if (what != NORM_ONLY) {
        bool fine = false;
        try {
            fine = apart(grads, dst, counts, tensors, what == CLIPPED);
        } catch (...) {
            return katsu_set_error(KATSU_ERR_ALLOC, "out of host memory");
        }
        KATSU_REQUIRE(fine, what == CLIPPED ? "outputs overlap each other or other gradients"
                                            : "weights overlap each other or gradients");
    }
    KATSU_TRY(katsu_bind(ctx));
    return live <= kFewTensors ? run<kFewTensors>(ctx, what, grads, dst, counts, tensors, lr, max_norm, norm)
                               : run<kMaxTensors>(ctx, what, grads, dst, counts, tensors, lr, max_norm, norm);
}

}  // namespace

extern "C" int32_t katsu_cuda_grad_norm(katsu_cuda_ctx *ctx, const float *const *grads, const size_t *counts, size_t tensors,
                                        float *norm) {
    return checked(ctx, NORM_ONLY, grads, nullptr, counts, tensors, 0.f, 0.f, norm);
}

extern "C" int32_t katsu_cuda_clip_grads(katsu_cuda_ctx *ctx, const float *const *grads, float *const *out,
                                         const size_t *counts, size_t tensors, float max_norm, float *norm) {
    return checked(ctx, CLIPPED, grads, out, counts, tensors, 0.f, max_norm, norm);
}

extern "C" int32_t katsu_cuda_sgd_step_clipped(katsu_cuda_ctx *ctx, float *const *weights, const float *const *grads,
                                               const size_t *counts, size_t tensors, float lr, float max_norm, float *norm) {
    return checked(ctx, STEPPED, grads, weights, counts, tensors, lr, max_norm, norm);
}
