// What a server does to logits before it picks a token from them, in one pass.
//
//   v = z / r or z r for tokens of the history      v -= f count + a for generated ones      v += biases      v = -inf if not allowed
//
// Bound: HBM, logits in (of allowed tokens) and out.  A block has a slice of a row: it counts the history's tokens of its slice in
// shared memory (whole numbers: atomics in any order give the same counts) while the slice's logits are on their way, and
// writes the slice once.  Tokens with biases, a few of a row, are written again behind it from the row's list in its order.
#include <math.h>

#include "common.cuh"
#include "launch.cuh"

namespace {

constexpr int kThreads = 256, kHeld = 8;
constexpr unsigned kSlice = 4 * kThreads * kHeld;  // tokens of a block
constexpr unsigned kInPrompt = 0x80000000u;        // beside the count of generated ones

struct Adjust {
    const float *logits, *repetition, *presence, *frequency, *bias;
    const int *history, *prompts, *lengths, *bias_tokens;
    const unsigned *allowed;
    float *out;
    unsigned rows, vocab, history_cols, biases, words, slices;
};

struct Penalties {
    float repetition, presence, frequency;
};

__device__ __forceinline__ float penalised(float v, unsigned seen, const Penalties &p) {
    if (seen == 0) return v;
    v = v > 0.f ? v / p.repetition : v * p.repetition;
    const unsigned count = seen & ~kInPrompt;
    return count ? v - fmaf(p.frequency, float(count), p.presence) : v;
}

__global__ void __launch_bounds__(kThreads) adjust_kernel(Adjust a) {
    extern __shared__ __align__(16) unsigned seen[];  // [kSlice + 4], behind it the row's biases
    const unsigned row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const float *z = a.logits + size_t(row) * a.vocab;
    float *out = a.out + size_t(row) * a.vocab;
    const unsigned *words = a.allowed ? a.allowed + size_t(row) * a.words : nullptr;
    // The slice's places are counted from the 16-byte boundary at or in front of the row.
    const unsigned lead = unsigned(reinterpret_cast<uintptr_t>(z) >> 2) & 3u, out_lead = unsigned(reinterpret_cast<uintptr_t>(out) >> 2) & 3u;
    const long long base = (long long)slice * kSlice - lead;  // token of the slice's place 0 (negative: none)
    // bit c: place 4 u + c is a token that is allowed
    auto allowed = [&](long long first) {
        unsigned bits = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const long long token = first + c;
            if (token < 0 || token >= a.vocab) continue;
            if (!words || (words[token >> 5] >> (token & 31) & 1u)) bits |= 1u << c;
        }
        return bits;
    };
    float4 v[kHeld];
    unsigned bits[kHeld];
#pragma unroll
    for (int q = 0; q < kHeld; ++q) {
        const long long first = base + 4ll * (q * kThreads + threadIdx.x);
        bits[q] = allowed(first);
        v[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (bits[q] == 0) continue;
        if (first >= 0 && first + 4 <= a.vocab) {
            v[q] = *reinterpret_cast<const float4 *>(z + first);
        } else {
            float one[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) one[c] = bits[q] >> c & 1u ? z[first + c] : 0.f;
            v[q] = make_float4(one[0], one[1], one[2], one[3]);
        }
    }
    Penalties p = {1.f, 0.f, 0.f};
    float *bias = reinterpret_cast<float *>(seen + kSlice), *bias_z = bias + a.biases;
    int *bias_tokens = reinterpret_cast<int *>(bias_z + a.biases);
    if (a.history) {
        for (unsigned i = threadIdx.x; i < kSlice / 4; i += kThreads) reinterpret_cast<uint4 *>(seen)[i] = make_uint4(0, 0, 0, 0);
        if (a.repetition) p.repetition = a.repetition[row];
        if (a.presence) p.presence = a.presence[row];
        if (a.frequency) p.frequency = a.frequency[row];
    }
    for (unsigned j = threadIdx.x; j < a.biases; j += kThreads) {
        const long long token = a.bias_tokens[size_t(row) * a.biases + j];
        const bool mine = token >= 0 && token < a.vocab && token >= base && token < base + kSlice;
        bias_tokens[j] = mine ? int(token) : -1;
        bias[j] = a.bias[size_t(row) * a.biases + j];
        bias_z[j] = mine ? z[token] : 0.f;
    }
    __syncthreads();
    if (a.history) {
        const unsigned length = a.lengths ? unsigned(min(max(a.lengths[row], 0), int(a.history_cols))) : a.history_cols;
        const unsigned prompt = a.prompts ? unsigned(min(max(a.prompts[row], 0), int(length))) : 0;
        const int *history = a.history + size_t(row) * a.history_cols;
#pragma unroll 8
        for (unsigned i = threadIdx.x; i < length; i += kThreads) {
            const int token = history[i];
            const long long place = token - base;
            if (token < 0 || unsigned(token) >= a.vocab || place < 0 || place >= kSlice) continue;
            if (i < prompt) atomicOr(&seen[place], kInPrompt);
            else atomicAdd(&seen[place], 1u);
        }
        __syncthreads();
    }
#pragma unroll
    for (int q = 0; q < kHeld; ++q) {
        const unsigned place = 4 * (q * kThreads + threadIdx.x);
        const long long first = base + place;
        if (first + 3 < 0 || first >= a.vocab) continue;
        float r[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
        if (a.history) {
            const uint4 s = *reinterpret_cast<const uint4 *>(seen + place);
            r[0] = penalised(r[0], s.x, p);
            r[1] = penalised(r[1], s.y, p);
            r[2] = penalised(r[2], s.z, p);
            r[3] = penalised(r[3], s.w, p);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (!(bits[q] >> c & 1u)) r[c] = -INFINITY;
        if (out_lead == lead && first >= 0 && first + 4 <= a.vocab) {
            *reinterpret_cast<float4 *>(out + first) = make_float4(r[0], r[1], r[2], r[3]);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (first + c >= 0 && first + c < a.vocab) out[first + c] = r[c];
        }
    }
    if (a.biases == 0) return;
    __syncthreads();
    for (unsigned j = threadIdx.x; j < a.biases; j += kThreads) {
        const int token = bias_tokens[j];
        if (token < 0 || (words && !(words[token >> 5] >> (token & 31) & 1u))) continue;
        bool first = true;
        float sum = 0.f;
        for (unsigned i = 0; i < a.biases; ++i) {
            if (bias_tokens[i] != token) continue;
            first = first && i >= j;
            sum += bias[i];
        }
        if (first) out[token] = (a.history ? penalised(bias_z[j], seen[token - base], p) : bias_z[j]) + sum;
    }
}

}  // namespace

extern "C" int32_t katsu_cuda_adjust_logits(katsu_cuda_ctx *ctx, const float *logits, const int32_t *history, const int32_t *prompts,
                                            const int32_t *lengths, const float *repetition, const float *presence,
                                            const float *frequency, const int32_t *bias_tokens, const float *bias,
                                            const uint32_t *allowed, float *out, size_t rows, size_t vocab, size_t history_cols,
                                            size_t biases) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_REQUIRE(rows <= 0x7fffffffu && vocab <= 0x7fffffffu && history_cols <= 0x7fffffffu, "rows, vocab and history_cols are below 2^31");
    KATSU_REQUIRE(biases <= KATSU_LOGITS_MAX_BIASES, "at most KATSU_LOGITS_MAX_BIASES biases of a row");
    if (rows == 0 || vocab == 0) return katsu_bind(ctx);
    KATSU_REQUIRE(logits != nullptr && out != nullptr, "logits or out is null");
    KATSU_REQUIRE(history != nullptr || history_cols == 0, "history is null");
    KATSU_REQUIRE(biases == 0 || (bias_tokens != nullptr && bias != nullptr), "bias_tokens or bias is null");
    const size_t bytes = 4 * rows * vocab, words = (vocab + 31) / 32;
    const struct {
        const void *p;
        size_t bytes;
    } in[] = {{logits, bytes}, {history, 4 * rows * history_cols}, {prompts, 4 * rows}, {lengths, 4 * rows}, {repetition, 4 * rows},
              {presence, 4 * rows}, {frequency, 4 * rows}, {bias_tokens, 4 * rows * biases}, {bias, 4 * rows * biases}, {allowed, 4 * rows * words}};
    for (const auto &i : in) {
        KATSU_REQUIRE(katsu_whole(i.p) && katsu_whole(out), "an address is not that of a whole element");
        KATSU_REQUIRE((i.p == logits && out == logits) || !katsu_overlap(out, bytes, i.p, i.bytes), "out overlaps an input");
    }
    Adjust a = {logits, repetition, presence, frequency, bias, history_cols ? history : nullptr, prompts, lengths, bias_tokens, allowed, out,
                unsigned(rows), unsigned(vocab), unsigned(history_cols), unsigned(biases), unsigned(words),
                unsigned((vocab + 3 + kSlice - 1) / kSlice)};
    const size_t blocks = rows * a.slices, smem = 4 * size_t(kSlice) + 12 * biases;
    if (blocks > 0x7fffffffu) return katsu_set_error(KATSU_ERR_UNSUPPORTED, "%zu rows of %zu logits in one call", rows, vocab);
    KATSU_TRY(katsu_bind(ctx));
    KATSU_LAUNCH(ctx, adjust_kernel, unsigned(blocks), kThreads, smem, a);
    return KATSU_OK;
}
