// What a server does to logits before it picks a token from them, in one pass.
//
//   v = z / r or z r for tokens of the history      v -= f count + a for generated ones      v += biases      v = -inf if not allowed
//
// Bound: HBM, logits in (of allowed tokens) and out; few rows: a chain of loads.  A block has a slice of a row: it counts the
// history's tokens of its slice in shared memory (whole numbers: atomics in any order give the same counts) while the slice's
// logits are on their way, and writes the slice once.  Tokens with biases, a few of a row, are written again behind it, by a token's
// first entry, with the sum over the row's list in its order.  In place only what changes is read and written.  512 x 100003: 65 us without
// a history, 6.3 TB/s; 64 x 131072 with histories of 4096 tokens 18 us, 14 without; under a grammar, with biases, 21.
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "launch.cuh"
#include "listed.cuh"

namespace {

constexpr int kThreads = 256, kBlocks = 4;  // blocks of an SM
constexpr int kHeld = 4, kAhead = 8;        // 16-byte accesses of a thread, and tokens of the history, on their way together
// Biases of a row above which a token's first entry is found by a table, in a kernel of its own: 64 x 131072 with histories of 4096 tokens,
// 150 biases 23 us by comparing all entries and 24 by a table, 300 39 and 31, 1000 211 and 62.
constexpr unsigned kCompared = 200;
constexpr unsigned kStep = 4 * kThreads, kMostSlice = 16 * kStep, kEdge = 8;  // kEdge: places for the edge

struct Adjust {
    const float *logits, *repetition, *presence, *frequency, *bias;
    const int *history, *prompts, *lengths, *bias_tokens;
    const unsigned *allowed;
    float *out;
    unsigned rows, vocab, history_cols, biases, words, slices;
    unsigned slice, places, masks;  // tokens of a block, a multiple of kStep; words of its places and of its part of the mask
    unsigned listed, firsts;        // words of a list of the biases, and of the table of their first entries
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

// TABLE: many biases
template <bool WIDE, bool TABLE>
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
    // A row is whole 16-byte units, cut into slices, and up to three tokens in front of the first and behind the last unit.  These, the
    // edge, go with the first slice: their places are behind the slice's.
    const unsigned head = min(a.vocab, (0u - unsigned(reinterpret_cast<uintptr_t>(z) >> 2)) & 3u), body = (a.vocab - head) & ~3u;
    const unsigned edge = slice ? 0 : a.vocab - body, begin = min(body, slice * a.slice), here = min(body - begin, a.slice);
    const unsigned base = head + begin;  // token of place 0; places 0 .. here - 1 are base, base + 1, ..
    auto edge_token = [&](unsigned i) { return i < head ? i : body + i; };
    auto place_of = [&](unsigned token) {  // ~0u: not of this block
        if (token - base < here) return token - base;
        if (token >= a.vocab || edge == 0 || (token >= head && token < head + body)) return ~0u;
        return a.slice + (token < head ? token : token - body);
    };
    // ---- what does not wait for anything: the slice's words of the mask, the history's first tokens ----
    unsigned *mask = seen + a.places;
    const unsigned word0 = base >> 5;
    if (words)
        for (unsigned i = threadIdx.x; i < a.slice / 32 + 2; i += kThreads) mask[i] = word0 + i < a.words ? words[word0 + i] : 0;
    const int *history = a.history ? a.history + size_t(row) * a.history_cols : nullptr;
    int first[kAhead];
    if (history)
#pragma unroll
        for (int q = 0; q < kAhead; ++q) first[q] = threadIdx.x + q * kThreads < a.history_cols ? history[threadIdx.x + q * kThreads] : -1;
    for (unsigned i = threadIdx.x; i < a.places / 4; i += kThreads) reinterpret_cast<uint4 *>(seen)[i] = make_uint4(0, 0, 0, 0);
    if (words) __syncthreads();
    // of the four tokens from place p on: bit c is that of place p + c
    auto allowed = [&](unsigned p) {
        if (!words) return 15u;
        const unsigned token = base + p, *at = mask + ((token >> 5) - word0);
        return __funnelshift_r(at[0], at[1], token & 31) & 15;
    };
    const float4 *units = reinterpret_cast<const float4 *>(z + base);
    float4 v[kHeld];
    unsigned bits[kHeld];
    auto ask = [&](unsigned from) {
#pragma unroll
        for (int q = 0; q < kHeld; ++q) {
            const unsigned p = from + q * kStep;
            bits[q] = p < here ? allowed(p) : 0;
            if (bits[q] && !in_place) v[q] = units[p / 4];
        }
    };
    ask(4 * threadIdx.x);
    // ---- the history's tokens and the biases of the slice ----
    float *bias = reinterpret_cast<float *>(mask + a.masks), *bias_z = bias + a.listed;
    int *bias_tokens = reinterpret_cast<int *>(bias_z + a.listed);
    const Listed tokens = {bias_tokens, bias_tokens + a.listed, bias_tokens + 2 * a.listed, a.firsts, a.biases};
    if (TABLE) {
        for (unsigned i = threadIdx.x; i < a.firsts; i += kThreads) tokens.table[i] = -1;
        if (threadIdx.x < a.listed - a.biases) bias_tokens[a.biases + threadIdx.x] = -1;
    }
    for (unsigned j = threadIdx.x; j < a.biases; j += kThreads) {
        const unsigned token = unsigned(a.bias_tokens[size_t(row) * a.biases + j]);
        const bool mine = place_of(token) != ~0u;
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
            for (int q = 0; q < kAhead; ++q) {
                const unsigned place = unsigned(token[q]) - base;
                if (place < here) P::count(seen, place, i + q * kThreads < prompt);
            }
            if (edge)
#pragma unroll
                for (int q = 0; q < kAhead; ++q) {
                    const unsigned t = unsigned(token[q]);
                    if (t < head || t - (head + body) < edge - head) P::count(seen, a.slice + (t < head ? t : t - body), i + q * kThreads < prompt);
                }
        }
    }
    if (history || a.biases) __syncthreads();
    if (TABLE)
        for (unsigned j = threadIdx.x; j < a.biases; j += kThreads) tokens.insert(j);
    // ---- the edge, and the slice ----
    auto is_allowed = [&](unsigned token) { return !words || (words[token >> 5] >> (token & 31) & 1u); };
    if (threadIdx.x < edge) {
        const unsigned token = edge_token(threadIdx.x);
        const float value = z[token];
        out[token] = !is_allowed(token) ? -INFINITY : history ? P::penalised(value, P::one(seen, place_of(token)), p) : value;
    }
    const bool whole = (reinterpret_cast<uintptr_t>(out + base) & 15u) == 0;
    for (unsigned from = 4 * threadIdx.x; from < here;) {
#pragma unroll
        for (int q = 0; q < kHeld; ++q) {
            const unsigned place = from + q * kStep, can = bits[q];
            if (place >= here) continue;
            uint4 s = make_uint4(0, 0, 0, 0);
            if (history) s = P::four(seen, place);
            const bool touched = (s.x | s.y | s.z | s.w) != 0;
            if (in_place) {
                if (can == 15 && !touched) continue;
                if (can) v[q] = units[place / 4];
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
            float *to = out + base + place;
            if (whole) {
                *reinterpret_cast<float4 *>(to) = v[q];
            } else {
                to[0] = v[q].x;
                to[1] = v[q].y;
                to[2] = v[q].z;
                to[3] = v[q].w;
            }
        }
        from += kHeld * kStep;
        ask(from);
    }
    if (a.biases == 0) return;
    __syncthreads();
    if (TABLE) {
        for (unsigned j = threadIdx.x; j < a.biases; j += kThreads) tokens.mark(j, bias[j]);
        __syncthreads();
    }
    for (unsigned j = threadIdx.x; j < a.biases; j += kThreads) {
        const int token = bias_tokens[j];
        if (token < 0 || !is_allowed(unsigned(token))) continue;
        bool first = true;
        float sum = 0.f;
        if (TABLE) {
            first = tokens.is_first(j);
            if (first) sum += tokens.sum(j, bias);
        } else {
            for (unsigned i = 0; i < a.biases; ++i) {
                if (bias_tokens[i] != token) continue;
                first = first && i >= j;
                sum += bias[i];
            }
        }
        if (first) out[token] = (history ? P::penalised(bias_z[j], P::one(seen, place_of(unsigned(token))), p) : bias_z[j]) + sum;
    }
}

template <bool WIDE, bool TABLE>
int32_t launch(katsu_cuda_ctx *ctx, Adjust a) {
    // One round of blocks, as every block looks at the row's whole history; slices are bounded by the shared memory for their places.
    const size_t resident = size_t(kBlocks) * ctx->num_sms, wanted = std::max<size_t>(1, resident / a.rows);
    a.slice = unsigned(std::min<size_t>(kMostSlice, katsu_div_up(katsu_div_up(a.vocab, wanted), kStep) * kStep));
    a.slices = unsigned(katsu_div_up(a.vocab, a.slice));
    a.places = !a.history ? 0 : WIDE ? a.slice + kEdge : (a.slice + kEdge) / 2;
    a.masks = a.allowed ? a.slice / 32 + (TABLE ? 4 : 2) : 0;
    a.listed = TABLE ? (a.biases + 3) / 4 * 4 : a.biases;  // (the table's tokens are read by 16 bytes)
    a.firsts = TABLE ? listed_places(a.biases) : 0;
    const size_t blocks = size_t(a.rows) * a.slices, smem = 4 * (size_t(a.places) + a.masks + (TABLE ? 4 : 3) * size_t(a.listed) + a.firsts);
    if (blocks > 0x7fffffffu) return katsu_set_error(KATSU_ERR_UNSUPPORTED, "%u rows of %u logits in one call", a.rows, a.vocab);
    KATSU_TRY(katsu_prepare_kernel(ctx, reinterpret_cast<const void *>(adjust_kernel<WIDE, TABLE>), smem, false));
    const size_t per_sm = std::min<size_t>(kBlocks, katsu_shared_per_sm() / (smem + 1024));
    a.waves = blocks > per_sm * ctx->num_sms;
    return katsu_launch(ctx, !a.waves, adjust_kernel<WIDE, TABLE>, unsigned(blocks), kThreads, smem, 1, a);
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
        // (out may be the logits' place: of this operand alone, whatever else is at their address)
        KATSU_REQUIRE((&i == in && out == logits) || !katsu_overlap(out, bytes, i.p, i.bytes), "out overlaps an input");
    }
    KATSU_TRY(katsu_bind(ctx));
    const Adjust a = {logits, repetition, presence, frequency, bias, history_cols ? history : nullptr, prompts, lengths, bias_tokens, allowed, out,
                      unsigned(rows), unsigned(vocab), unsigned(history_cols), unsigned(biases), unsigned(words), 0, 0, 0, 0, 0, 0, 0};
    const bool wide = history_cols >= 1 << 15;
    if (biases > kCompared) return wide ? launch<true, true>(ctx, a) : launch<false, true>(ctx, a);
    return wide ? launch<true, false>(ctx, a) : launch<false, false>(ctx, a);
}
