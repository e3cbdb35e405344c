// What a server does to logits before it picks a token from them, in one pass.
//
//   v = z / r or z r for tokens of the history      v -= f count + a for generated ones      v += biases      v = -inf if not allowed
//
// Bound: HBM, logits in (of allowed tokens) and out; few rows: a chain of loads.  A block has a slice of a row: it counts the
// history's tokens of its slice in shared memory (whole numbers: atomics in any order give the same counts) while the slice's
// logits are on their way, and writes the slice once.  Tokens with biases, a few of a row, are written again behind it from the
// row's list in its order.  In place only what changes is read and written.
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "launch.cuh"

namespace {

constexpr int kThreads = 256, kBlocks = 4;  // blocks of an SM
constexpr int kHeld = 4, kAhead = 8;        // 16-byte accesses of a thread, and tokens of the history, on their way together
constexpr unsigned kStep = 4 * kThreads, kMostSlice = 16 * kStep;

struct Adjust {
    const float *logits, *repetition, *presence, *frequency, *bias;
    const int *history, *prompts, *lengths, *bias_tokens;
    const unsigned *allowed;
    float *out;
    unsigned rows, vocab, history_cols, biases, words, slices;
    unsigned slice, places, masks;  // tokens of a block, a multiple of kStep; words of its places and of its part of the mask
    int waves;
};

struct Penalties {
    float repetition, presence, frequency;
};

// A token's place: how often it is in the generated part, and a bit above for the prompt.  Two places share a word where the history
// has less than 2^15 tokens.
template <bool WIDE>
struct Place {
    static constexpr unsigned kPrompt = WIDE ? 0x80000000u : 0x8000u;
    static __device__ __forceinline__ void count(unsigned *seen, unsigned place, bool prompt) {
        if (WIDE) {
            if (prompt) atomicOr(&seen[place], kPrompt);
            else atomicAdd(&seen[place], 1u);
        } else {
            const unsigned up = 16 * (place & 1);
            if (prompt) atomicOr(&seen[place >> 1], kPrompt << up);
            else atomicAdd(&seen[place >> 1], 1u << up);
        }
    }
    static __device__ __forceinline__ unsigned one(const unsigned *seen, unsigned place) {
        return WIDE ? seen[place] : seen[place >> 1] >> (16 * (place & 1)) & 0xffffu;
    }
    // four places from a multiple of four on
    static __device__ __forceinline__ uint4 four(const unsigned *seen, unsigned place) {
        if (WIDE) return *reinterpret_cast<const uint4 *>(seen + place);
        const uint2 two = *reinterpret_cast<const uint2 *>(seen + place / 2);
        return make_uint4(two.x & 0xffffu, two.x >> 16, two.y & 0xffffu, two.y >> 16);
    }
    static __device__ __forceinline__ float penalised(float v, unsigned seen, const Penalties &p) {
        if (seen == 0) return v;
        v = v > 0.f ? v / p.repetition : v * p.repetition;
        const unsigned count = seen & ~kPrompt;
        return count ? v - fmaf(p.frequency, float(count), p.presence) : v;
    }
};

template <bool WIDE>
__global__ void __launch_bounds__(kThreads, kBlocks) adjust_kernel(Adjust a) {
    using P = Place<WIDE>;
    extern __shared__ __align__(16) unsigned seen[];  // the places; the slice's words of the mask; the row's biases
    if (!a.waves) launch_next();
    launch_wait();
    const unsigned row = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const float *z = a.logits + size_t(row) * a.vocab;
    float *out = a.out + size_t(row) * a.vocab;
    const bool in_place = z == out;
    const unsigned *words = a.allowed ? a.allowed + size_t(row) * a.words : nullptr;
    // The slice's places are counted from the 16-byte boundary at or in front of the row: base is the token of place 0.  Tokens are
    // taken modulo 2^32, so that the up to three places in front of the row are numbers above the vocabulary.
    const unsigned lead = unsigned(reinterpret_cast<uintptr_t>(z) >> 2) & 3u, base = slice * a.slice - lead;
    const bool inside = base < a.vocab && a.vocab - base >= a.slice;  // (of all the slice's places)
    const bool whole = (unsigned(reinterpret_cast<uintptr_t>(out) >> 2) & 3u) == lead;
    // ---- what does not wait for anything: the slice's words of the mask and the history's first tokens ----
    unsigned *mask = seen + a.places;
    const unsigned word0 = base < a.vocab ? base >> 5 : 0;
    if (words)
        for (unsigned i = threadIdx.x; i < a.slice / 32 + 2; i += kThreads) mask[i] = word0 + i < a.words ? words[word0 + i] : 0;
    const int *history = a.history ? a.history + size_t(row) * a.history_cols : nullptr;
    int first[kAhead];
    if (history)
#pragma unroll
        for (int q = 0; q < kAhead; ++q) first[q] = threadIdx.x + q * kThreads < a.history_cols ? history[threadIdx.x + q * kThreads] : -1;
    for (unsigned i = threadIdx.x; i < a.places / 4; i += kThreads) reinterpret_cast<uint4 *>(seen)[i] = make_uint4(0, 0, 0, 0);
    if (words) __syncthreads();
    // which of an access's tokens are allowed: bit c of token + c
    auto allowed = [&](unsigned token) {
        unsigned bits = 15;
        if (!inside) {
            bits = 0;
#pragma unroll
            for (unsigned c = 0; c < 4; ++c)
                if (token + c < a.vocab && (!words || (mask[((token + c) >> 5) - word0] >> ((token + c) & 31) & 1u))) bits |= 1u << c;
        } else if (words) {
            const unsigned *at = mask + ((token >> 5) - word0);
            bits = __funnelshift_r(at[0], at[1], token & 31) & 15;
        }
        return bits;
    };
    auto fetch = [&](unsigned token, unsigned bits) {
        if (bits == 0) return make_float4(0.f, 0.f, 0.f, 0.f);
        if (inside) return *reinterpret_cast<const float4 *>(z + token);
        return make_float4(bits & 1 ? z[token] : 0.f, bits & 2 ? z[token + 1] : 0.f, bits & 4 ? z[token + 2] : 0.f, bits & 8 ? z[token + 3] : 0.f);
    };
    float4 v[kHeld];
    unsigned bits[kHeld];
    auto ask = [&](unsigned from) {
#pragma unroll
        for (int q = 0; q < kHeld; ++q) {
            const unsigned place = from + q * kStep;
            bits[q] = place < a.slice ? allowed(base + place) : 0;
            if (!in_place) v[q] = fetch(base + place, bits[q]);
        }
    };
    ask(4 * threadIdx.x);
    // ---- the history's tokens and the biases of the slice ----
    float *bias = reinterpret_cast<float *>(mask + a.masks), *bias_z = bias + a.biases;
    int *bias_tokens = reinterpret_cast<int *>(bias_z + a.biases);
    for (unsigned j = threadIdx.x; j < a.biases; j += kThreads) {
        const unsigned token = unsigned(a.bias_tokens[size_t(row) * a.biases + j]);
        const bool mine = token < a.vocab && token - base < a.slice;
        bias_tokens[j] = mine ? int(token) : -1;
        bias[j] = a.bias[size_t(row) * a.biases + j];
        bias_z[j] = mine ? z[token] : 0.f;
    }
    Penalties p = {1.f, 0.f, 0.f};
    if (history) {
        const unsigned length = a.lengths ? unsigned(min(max(a.lengths[row], 0), int(a.history_cols))) : a.history_cols;
        const unsigned prompt = a.prompts ? unsigned(min(max(a.prompts[row], 0), int(length))) : 0;
        if (a.repetition) p.repetition = a.repetition[row];
        if (a.presence) p.presence = a.presence[row];
        if (a.frequency) p.frequency = a.frequency[row];
        __syncthreads();
        for (unsigned i = threadIdx.x; i < length; i += kAhead * kThreads) {
            int token[kAhead];
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const unsigned at = i + q * kThreads;
                token[q] = at >= length ? -1 : i == threadIdx.x ? first[q] : history[at];
            }
#pragma unroll
            for (int q = 0; q < kAhead; ++q)
                if (unsigned(token[q]) < a.vocab && unsigned(token[q]) - base < a.slice) P::count(seen, unsigned(token[q]) - base, i + q * kThreads < prompt);
        }
    }
    if (history || a.biases) __syncthreads();
    // ---- the slice ----
    for (unsigned from = 4 * threadIdx.x;;) {
#pragma unroll
        for (int q = 0; q < kHeld; ++q) {
            const unsigned place = from + q * kStep, token = base + place, can = bits[q];
            if (place >= a.slice) continue;
            uint4 s = make_uint4(0, 0, 0, 0);
            if (history) s = P::four(seen, place);
            const bool touched = (s.x | s.y | s.z | s.w) != 0;
            if (in_place) {
                if (can == 15 && !touched) continue;
                v[q] = fetch(token, can);
            }
            if (touched) {
                v[q].x = P::penalised(v[q].x, s.x, p);
                v[q].y = P::penalised(v[q].y, s.y, p);
                v[q].z = P::penalised(v[q].z, s.z, p);
                v[q].w = P::penalised(v[q].w, s.w, p);
            }
            if (!(can & 1)) v[q].x = -INFINITY;
            if (!(can & 2)) v[q].y = -INFINITY;
            if (!(can & 4)) v[q].z = -INFINITY;
            if (!(can & 8)) v[q].w = -INFINITY;
            if (inside && whole) {
                *reinterpret_cast<float4 *>(out + token) = v[q];
            } else {
                if (token < a.vocab) out[token] = v[q].x;
                if (token + 1 < a.vocab) out[token + 1] = v[q].y;
                if (token + 2 < a.vocab) out[token + 2] = v[q].z;
                if (token + 3 < a.vocab) out[token + 3] = v[q].w;
            }
        }
        from += kHeld * kStep;
        if (from >= a.slice) break;
        ask(from);
    }
    if (a.biases == 0) return;
    __syncthreads();
    for (unsigned j = threadIdx.x; j < a.biases; j += kThreads) {
        const int token = bias_tokens[j];
        if (token < 0 || (words && !(mask[(token >> 5) - word0] >> (token & 31) & 1u))) continue;
        bool first = true;
        float sum = 0.f;
        for (unsigned i = 0; i < a.biases; ++i) {
            if (bias_tokens[i] != token) continue;
            first = first && i >= j;
            sum += bias[i];
        }
        if (first) out[token] = (history ? P::penalised(bias_z[j], P::one(seen, unsigned(token) - base), p) : bias_z[j]) + sum;
    }
}

template <bool WIDE>
int32_t launch(katsu_cuda_ctx *ctx, Adjust a) {
    // One round of blocks, as every block looks at the row's whole history; slices are bounded by the shared memory for their places.
    const size_t places = size_t(a.vocab) + 3, resident = size_t(kBlocks) * ctx->num_sms, wanted = std::max<size_t>(1, resident / a.rows);
    a.slice = unsigned(std::min<size_t>(kMostSlice, katsu_div_up(katsu_div_up(places, wanted), kStep) * kStep));
    a.slices = unsigned(katsu_div_up(places, a.slice));
    a.places = !a.history ? 0 : WIDE ? a.slice : a.slice / 2;
    a.masks = a.allowed ? a.slice / 32 + 2 : 0;
    const size_t blocks = size_t(a.rows) * a.slices, smem = 4 * (size_t(a.places) + a.masks + 3 * size_t(a.biases));
    if (blocks > 0x7fffffffu) return katsu_set_error(KATSU_ERR_UNSUPPORTED, "%u rows of %u logits in one call", a.rows, a.vocab);
    KATSU_TRY(katsu_prepare_kernel(ctx, reinterpret_cast<const void *>(adjust_kernel<WIDE>), smem, false));
    const size_t per_sm = std::min<size_t>(kBlocks, katsu_shared_per_sm() / (smem + 1024));
    a.waves = blocks > per_sm * ctx->num_sms;
    return katsu_launch(ctx, !a.waves, adjust_kernel<WIDE>, unsigned(blocks), kThreads, smem, 1, a);
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
    KATSU_TRY(katsu_bind(ctx));
    const Adjust a = {logits, repetition, presence, frequency, bias, history_cols ? history : nullptr, prompts, lengths, bias_tokens, allowed, out,
                      unsigned(rows), unsigned(vocab), unsigned(history_cols), unsigned(biases), unsigned(words), 0, 0, 0, 0, 0};
    const bool wide = history_cols >= 1 << 15;
    return wide ? launch<true>(ctx, a) : launch<false>(ctx, a);
}
