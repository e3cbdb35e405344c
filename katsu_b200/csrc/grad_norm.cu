// The norm over all gradients of a step, clipping by it, and the SGD step with clipped gradients.
//
//   norm = sqrt(sum over all tensors of g^2)      c = max_norm / norm where that is below 1      g' = c g      w -= lr (c g)
//
// Two launches whatever the number of tensors (one more pair for every 512): the first leaves a partial sum of squares a
// block, the blocks of the second fold these for themselves and then scale or step.  The addresses travel as a kernel
// parameter, so nothing on the host has to outlive the call and a captured call keeps them.
//
// Squares are summed in 64 bits: 1e-30 and 1e30 neither vanish nor overflow, the sum of 1e9 values keeps more bits than the
// f32 result shows, and a sum that is not finite means exactly that a gradient is not.  It costs nothing beside the loads: a
// conversion and a multiply-add a value, 16 and 64 lanes a clock and SM, where the memory brings 6 values.
#include <math.h>

#include <algorithm>
#include <new>
#include <vector>

#include "common.cuh"
#include "launch.cuh"

namespace {

constexpr int kThreads = 256;
constexpr unsigned kChunk = 4096;  // values a block takes at a time: four 16-byte loads a thread
constexpr int kMaxTensors = 512;   // a launch (14 KiB of parameters)
constexpr int kFewTensors = 32;    // (1 KiB: the launch of a large parameter block takes longer)

// Tensors of one launch.  Chunk c of a tensor has the values whose place behind the 16-byte boundary at or in front of the
// tensor is c * kChunk .. c * kChunk + kChunk - 1, so that 16-byte accesses fit tensors at any address.
template <int N>
struct Tensors {
    const float *src[N];
    float *dst[N];
    unsigned long long count[N];
    unsigned first[N + 1];  // chunks in front of the tensor
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

template <int N>
__device__ __forceinline__ int tensor_of(const Tensors<N> &t, unsigned chunk) {
    int lo = 0, hi = t.tensors - 1;  // the last tensor whose first chunk is not behind this one (empty ones have none)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ unsigned lead_of(const float *p) { return unsigned(reinterpret_cast<uintptr_t>(p) >> 2) & 3u; }

// partial[block] = the block's sum of squares.
template <int N>
__global__ void __launch_bounds__(kThreads) squares_kernel(const __grid_constant__ Tensors<N> t, double *partial) {
    launch_next();
    launch_wait();
    double acc = 0.0;
    for (unsigned chunk = blockIdx.x; chunk < t.first[t.tensors]; chunk += gridDim.x) {
        const int i = tensor_of(t, chunk);
        const float *src = t.src[i];
        const unsigned lead = lead_of(src);
        const float *base = src - lead;
        const unsigned long long begin = (unsigned long long)(chunk - t.first[i]) * kChunk, end = lead + t.count[i];
        float4 v[kChunk / 4 / kThreads];
#pragma unroll
        for (int j = 0; j < int(kChunk / 4 / kThreads); ++j) {
            const unsigned long long a = begin + 4ull * (threadIdx.x + j * kThreads);
            if (a >= lead && a + 4 <= end) {
                v[j] = __ldg(reinterpret_cast<const float4 *>(base + a));
            } else {
                v[j].x = a >= lead && a < end ? __ldg(base + a) : 0.f;
                v[j].y = a + 1 >= lead && a + 1 < end ? __ldg(base + a + 1) : 0.f;
                v[j].z = a + 2 >= lead && a + 2 < end ? __ldg(base + a + 2) : 0.f;
                v[j].w = a + 3 >= lead && a + 3 < end ? __ldg(base + a + 3) : 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < int(kChunk / 4 / kThreads); ++j) {
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
__device__ __forceinline__ double fold(const double *partial, int parts) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < parts; i += kThreads) acc += __ldcg(partial + i);
    __shared__ double sh[kThreads / 32];
    return block_sum(acc, sh);
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double *partial, int parts, float *norm) {
    launch_next();
    launch_wait();
    const double sum = fold(partial, parts);
    if (threadIdx.x == 0) norm[0] = (float)sqrt(sum);
}

// g and the product are rounded as katsu_cuda_clip_grads followed by katsu_cuda_sgd_step round them.
template <Apply OP>
__device__ __forceinline__ float applied(float g, float w, float c, float lr) {
    const float clipped = __fmul_rn(g, c);
    return OP == CLIP ? clipped : w - __fmul_rn(lr, clipped);
}

template <Apply OP, int N>
__global__ void __launch_bounds__(kThreads) apply_kernel(const __grid_constant__ Tensors<N> t, const double *partial, int parts,
                                                         float max_norm, float lr, float *norm) {
    launch_next();
    launch_wait();
    const double sum = fold(partial, parts), total = sqrt(sum);
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)total;
    const bool finite = isfinite(sum);
    if (OP == STEP && !finite) return;
    const float c = finite && total > (double)max_norm ? (float)((double)max_norm / total) : 1.f;
    const unsigned chunks = t.first[t.tensors];
    // from the last chunk to the first: what the pass over the squares has read last is still in L2
    for (unsigned q = blockIdx.x; q < chunks; q += gridDim.x) {
        const unsigned chunk = chunks - 1 - q;
        const int i = tensor_of(t, chunk);
        const float *src = t.src[i];
        float *dst = t.dst[i];
        if (OP == CLIP && c == 1.f && src == dst) continue;
        const unsigned lead = lead_of(src);
        const unsigned long long begin = (unsigned long long)(chunk - t.first[i]) * kChunk, end = lead + t.count[i];
        const float *sb = src - lead;
        float *db = dst - lead;
        if (lead_of(dst) == lead) {
            constexpr int loads = kChunk / 4 / kThreads;
            float4 g[loads], w[loads];
#pragma unroll
            for (int j = 0; j < loads; ++j) {
                const unsigned long long a = begin + 4ull * (threadIdx.x + j * kThreads);
                if (a >= lead && a + 4 <= end) {
                    g[j] = *reinterpret_cast<const float4 *>(sb + a);
                    if (OP == STEP) w[j] = *reinterpret_cast<const float4 *>(db + a);
                }
            }
#pragma unroll
            for (int j = 0; j < loads; ++j) {
                const unsigned long long a = begin + 4ull * (threadIdx.x + j * kThreads);
                if (a >= lead && a + 4 <= end) {
                    float4 o;
                    o.x = applied<OP>(g[j].x, OP == STEP ? w[j].x : 0.f, c, lr);
                    o.y = applied<OP>(g[j].y, OP == STEP ? w[j].y : 0.f, c, lr);
                    o.z = applied<OP>(g[j].z, OP == STEP ? w[j].z : 0.f, c, lr);
                    o.w = applied<OP>(g[j].w, OP == STEP ? w[j].w : 0.f, c, lr);
                    *reinterpret_cast<float4 *>(db + a) = o;
                } else {
                    for (unsigned long long b = a; b < a + 4; ++b)
                        if (b >= lead && b < end) db[b] = applied<OP>(sb[b], OP == STEP ? db[b] : 0.f, c, lr);
                }
            }
        } else {
            const unsigned long long last = begin + kChunk < end ? begin + kChunk : end;
            for (unsigned long long b = begin + threadIdx.x; b < last; b += kThreads)
                if (b >= lead) db[b] = applied<OP>(sb[b], OP == STEP ? db[b] : 0.f, c, lr);
        }
    }
}

template <int N>
size_t take(Tensors<N> *t, const float *const *src, float *const *dst, const size_t *counts, size_t from, size_t tensors) {
    int k = 0;
    unsigned long long chunks = 0;
    size_t i = from;
    for (; i < tensors && k < N; ++i) {
        if (counts[i] == 0) continue;
        const unsigned long long lead = (reinterpret_cast<uintptr_t>(src[i]) >> 2) & 3u;
        const unsigned long long more = (lead + counts[i] + kChunk - 1) / kChunk;
        if (k > 0 && chunks + more > 0xf0000000ull) break;
        t->src[k] = src[i];
        t->dst[k] = dst ? dst[i] : nullptr;
        t->count[k] = counts[i];
        t->first[k] = (unsigned)chunks;
        chunks += more;
        t->first[++k] = (unsigned)chunks;
    }
    t->tensors = k;
    return i;
}

unsigned blocks_for(const katsu_cuda_ctx *ctx, unsigned chunks) {
    const unsigned most = unsigned(ctx->num_sms) * 8;
    return chunks < most ? chunks : most;
}

enum What { NORM_ONLY, CLIPPED, STEPPED };

template <int N>
int32_t run(katsu_cuda_ctx *ctx, What what, const float *const *grads, float *const *dst, const size_t *counts, size_t tensors,
            float lr, float max_norm, float *norm) {
    static thread_local Tensors<N> t;  // (too large for some hosts' stacks)
    const size_t most = (size_t)ctx->num_sms * 8;
    size_t launches = 0;
    for (size_t i = 0; i < tensors; ++launches) i = take(&t, grads, dst, counts, i, tensors);
    float *scratch = nullptr;
    KATSU_TRY(katsu_scratch(ctx, (launches + 1) * most * 2, &scratch));
    double *partial = reinterpret_cast<double *>(scratch);
    KATSU_TRY(katsu_prepare_kernel(ctx, (const void *)squares_kernel<N>, 0));
    int parts = 0;
    for (size_t i = 0; i < tensors;) {
        i = take(&t, grads, dst, counts, i, tensors);
        if (t.tensors == 0) break;
        const unsigned blocks = blocks_for(ctx, t.first[t.tensors]);
        KATSU_TRY(katsu_launch_chained(ctx, squares_kernel<N>, blocks, kThreads, 0, 1, t, partial + parts));
        parts += (int)blocks;
    }
    if (what == NORM_ONLY || parts == 0) {
        KATSU_TRY(katsu_prepare_kernel(ctx, (const void *)norm_kernel, 0));
        return katsu_launch_chained(ctx, norm_kernel, 1, kThreads, 0, 1, partial, parts, norm);
    }
    auto kernel = what == CLIPPED ? apply_kernel<CLIP, N> : apply_kernel<STEP, N>;
    KATSU_TRY(katsu_prepare_kernel(ctx, (const void *)kernel, 0));
    for (size_t i = 0; i < tensors;) {
        const bool first = i == 0;
        i = take(&t, grads, dst, counts, i, tensors);
        if (t.tensors == 0) break;
        const unsigned blocks = blocks_for(ctx, t.first[t.tensors]);
        KATSU_TRY(katsu_launch_chained(ctx, kernel, blocks, kThreads, 0, 1, t, partial, parts, max_norm, lr, first ? norm : nullptr));
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
    KATSU_REQUIRE(tensors == 0 || (grads != nullptr && counts != nullptr), "null array of gradients or counts");
    KATSU_REQUIRE(tensors == 0 || what == NORM_ONLY || dst != nullptr, "null array of outputs or weights");
    KATSU_REQUIRE(what == NORM_ONLY || max_norm >= 0.f, "max_norm must be 0 or more");
    size_t live = 0;
    const auto holds_norm = [&](const float *p, size_t count) { return norm + 1 > p && norm < p + count; };
    for (size_t i = 0; i < tensors; ++i) {
        if (counts[i] == 0) continue;
        KATSU_REQUIRE(counts[i] < (size_t(1) << 43), "count out of range");
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
