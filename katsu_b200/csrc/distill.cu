// Loss of logits against a teacher's top logits and against labels, and its gradient.
//
//   p = softmax(t / T) over the listed entries      q = softmax(z / T), s = softmax(z) over the vocabulary
//   loss = w (soft T^2 sum_j p_j (log p_j - log q_idx(j)) - hard log s_label)
//   dz   = g w (soft T (q - p) + hard (s - [v = label]))
//
// Bound: HBM, z once and dz once (4096 x 32768, T = 2, labels too: loss 82 us, 5.9 TB/s; with the gradient 180 us, 5.7 TB/s; L2 has
// every row of the gradient's second reading).  Short or few rows: a block's chain of loads, votes and exchanges, 4 to 6 us.
//
// Blocks stream their row, threads with sums of their own (a largest value, sums of exponentials counted from it), four 16-byte loads
// on their way and five blocks of 256 threads to an SM: rows held in the registers of two blocks of 512 threads took five times as
// long, as nothing was on its way while a block exchanged its sums.  Threads, warps, blocks and the blocks of a cluster join their sums
// in a tree.  A warp beside the others goes through the row's list and label, whose loads follow each other.  The gradient reads the
// row again, from L2: threads and blocks are chosen so that the rows of all resident blocks fit there.  The gradient of listed tokens,
// a few of a row, is written again behind the row's, by a token's first entry, which a table in shared memory finds, from a sum over the
// list in its order: the same bits every time (comparing all entries took 1631 us of 4096 x 32768 with 1000 of them, now 300).
#include <float.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "launch.cuh"
#include "listed.cuh"
#include "sm100_pair.cuh"

namespace {

constexpr int kHeld = 4;  // 16-byte accesses of a thread on their way together
constexpr int kMostCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;

struct Distill {
    const float *logits, *teacher, *weight, *g;
    const int *index, *labels;
    float *loss, *dlogits;
    float temperature, soft, hard;
    float c0, c1;  // log2(e) / T and log2(e)
    unsigned rows, vocab, top, blocks;  // blocks of a row
    unsigned places;  // of the gradient's table of listed tokens, a power of two
    int accumulate, waves;
};

struct Sums {
    float m, s0, s1;  // largest value; sums of exp((z - m) / T) and of exp(z - m)
};

// A warp or block without a value above -infinity counts from the lowest number, which leaves its sums 0.
__device__ __forceinline__ float base_of(float m) { return fmaxf(m, -FLT_MAX); }
// 2^(d c), zero where that is no normal number
__device__ __forceinline__ float ex(float d, float c) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * c));
    return r;
}

template <bool TWO>
__device__ __forceinline__ Sums join(const Distill &a, Sums x, Sums y) {
    Sums r;
    r.m = fmaxf(x.m, y.m);
    const float b = base_of(r.m), dx = base_of(x.m) - b, dy = base_of(y.m) - b;
    r.s0 = x.s0 * ex(dx, a.c0) + y.s0 * ex(dy, a.c0);
    r.s1 = TWO ? x.s1 * ex(dx, a.c1) + y.s1 * ex(dy, a.c1) : 0.f;
    return r;
}

// Joins those of LANES neighbouring lanes: the largest value first, every lane's sums counted from it, then their sum.
template <bool TWO, int LANES>
__device__ __forceinline__ Sums join_lanes(const Distill &a, Sums x) {
    float most = x.m;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float d = base_of(x.m) - base_of(most);
    x.m = most;
    x.s0 *= ex(d, a.c0);
    if (TWO) x.s1 *= ex(d, a.c1);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        x.s0 += __shfl_xor_sync(0xffffffffu, x.s0, o);
        if (TWO) x.s1 += __shfl_xor_sync(0xffffffffu, x.s1, o);
    }
    return x;
}

__device__ __forceinline__ float largest_of_warp(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float sum_of_warp(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ double sum_of_warp(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The row's entries and, as the last one, its label: in shared memory, written by the warp behind the others.
struct Entries {
    int *token;  // -1 where it is none
    float *e;    // exp((t - largest t) / T), 0 for the label
    float *z;    // the token's logit
    float *t;    // t - largest t
};
// Entries that the list's warp puts into the table alone, while the others go through the row; longer lists all threads behind it.  4096 x
// 32768 with its gradient: 200 entries 196 us alone, 209 by all; 400 entries 230 and 225, and of 64 rows 18 and 13.
constexpr unsigned kAlone = 256;

// Copies 4 bytes to shared memory; wait_copies() waits for those of the thread.
__device__ __forceinline__ void copy_word(void *to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A row as whole 16-byte units, and up to three values in front of the first and behind the last one, which the first block of
// the row takes, a value a thread.
struct Row {
    unsigned head, units, edge;  // values in front; units; values in front and behind
    unsigned begin, end;         // the block's units

    __device__ Row(const float *z, unsigned vocab, unsigned rank, unsigned blocks) {
        head = min(vocab, (0u - unsigned(reinterpret_cast<uintptr_t>(z) >> 2)) & 3u);
        units = (vocab - head) / 4;
        edge = rank ? 0 : vocab - 4 * units;
        const unsigned share = (units + blocks - 1) / blocks;
        begin = min(units, rank * share);
        end = min(units, begin + share);
    }
    __device__ unsigned edge_token(unsigned i) const { return i < head ? i : 4 * units + i; }
    __device__ bool has(unsigned token) const {
        const unsigned place = token - head;
        if (token >= head && place < 4 * units) return place >= 4 * begin && place < 4 * end;
        return edge != 0;
    }
};

// Blocks of an SM: five of 256 threads, which have 40 registers each; 17, 10 and 3 of 64, 128 and 512, which are 51 warps, three more than
// fit with 40, and so have 32: the gradient with both sums then keeps 68 bytes a thread in local memory, the loss up to 28.  More warps are
// worth that.  Two blocks of 512 threads, with 56 registers and nothing in local memory, take 194 us for 4096 x 32768 instead of 180, 206
// instead of 189 for 2000 x 65536; 9 of 128 and 16 of 64 threads with 40 registers 41 instead of 38 for 8192 x 1003, 227 instead of 213 for
// 100 000 x 50.
constexpr int blocks_of_sm(int threads) { return 65536 / ((threads + 32) * 40); }

// THREADS threads go through the row, the warp behind them through its entries.  GRAD: writes the gradient (and the loss where it is
// asked for).  TWO: sums at the temperature and at 1; otherwise one set of sums is both.
template <int THREADS, bool GRAD, bool TWO>
__global__ void __launch_bounds__(THREADS + 32, blocks_of_sm(THREADS)) distill_kernel(Distill a) {
    extern __shared__ __align__(16) float dynamic[];
    __shared__ Sums of_warp[THREADS / 32];
    __shared__ Sums of_block[kMostCluster];
    __shared__ float teacher_sum;
    if (!a.waves) launch_next();
    launch_wait();
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned row = blockIdx.x / a.blocks, rank = blockIdx.x % a.blocks;
    const float weight = a.weight ? a.weight[row] : 1.f, of_row = GRAD && a.g ? a.g[row] : 1.f;
    const float *z = a.logits + size_t(row) * a.vocab;
    float *dz = GRAD ? a.dlogits + size_t(row) * a.vocab : nullptr;
    const Row part(z, a.vocab, rank, a.blocks);
    const float4 *body = reinterpret_cast<const float4 *>(z + part.head);
    auto zeros = [&] {
        for (unsigned v = part.head + 4 * part.begin + threadIdx.x; v < part.head + 4 * part.end; v += THREADS + 32) dz[v] = 0.f;
        if (threadIdx.x < part.edge) dz[part.edge_token(threadIdx.x)] = 0.f;
    };
    if (weight == 0.f) {  // (all blocks of the row)
        if (GRAD && !a.accumulate) zeros();
        if (a.loss && rank == 0 && threadIdx.x == 0) a.loss[row] = 0.f;
        return;
    }
    if (a.blocks > 1) sm100::cluster_arrive();
    const unsigned listed = a.top + 1, array = (listed + 3) & ~3u;  // (tokens are read by 16 bytes)
    int *const ints = reinterpret_cast<int *>(dynamic);
    const Entries entries = {ints, dynamic + array, dynamic + 2 * array, dynamic + 3 * array};
    const Listed tokens = {ints, ints + 4 * array, ints + 5 * array, a.places, listed};  // (the gradient's)
    if (warp == THREADS / 32) {
        // ---- the teacher's entries ----
        const int label = a.labels ? a.labels[row] : -1;
        // (copies, all on their way together: with 1000 entries the loss of 4096 x 32768 took 149 us by loads, 119 by copies)
        for (unsigned j = lane; j < a.top; j += 32) {
            copy_word(entries.token + j, a.index + size_t(row) * a.top + j);
            copy_word(entries.t + j, a.teacher + size_t(row) * a.top + j);
        }
        if (GRAD)
            for (unsigned i = lane; i < a.places; i += 32) tokens.table[i] = -1;
        wait_copies();
        float most = -INFINITY;
        for (unsigned j = lane; j < a.top; j += 32) {
            const int token = entries.token[j];
            if (unsigned(token) < a.vocab) {
                copy_word(entries.z + j, z + token);
                most = fmaxf(most, entries.t[j]);
            } else {
                entries.token[j] = -1;
                entries.z[j] = 0.f;
                entries.t[j] = -INFINITY;
            }
        }
        most = base_of(largest_of_warp(most));
        float sum = 0.f;
#pragma unroll 2
        for (unsigned j = lane; j < a.top; j += 32) {
            const float t = entries.t[j] - most, e = entries.token[j] >= 0 ? expf(t / a.temperature) : 0.f;
            entries.t[j] = t;
            entries.e[j] = e;
            sum += e;
        }
        sum = sum_of_warp(sum);
        if (lane == 0) {
            const bool there = unsigned(label) < a.vocab;
            entries.token[a.top] = there ? label : -1;
            entries.z[a.top] = there ? z[label] : 0.f;
            entries.e[a.top] = 0.f;
            teacher_sum = sum;
        }
        if (lane > 0 && a.top + lane < array) entries.token[a.top + lane] = -1;
        wait_copies();
        if (GRAD && a.top <= kAlone) {
            __syncwarp();
            for (unsigned j = lane; j < listed; j += 32) tokens.insert(j);
            __syncwarp();
            for (unsigned j = lane; j < listed; j += 32) tokens.mark(j, entries.e[j]);
        }
    } else {
        // ---- largest value and sums of the row: a thread's own, then the warp's ----
        Sums s = {threadIdx.x < part.edge ? z[part.edge_token(threadIdx.x)] : -INFINITY, 0.f, 0.f};
        s.s0 = s.s1 = ex(s.m - base_of(s.m), a.c0);
        auto take = [&](const float4 (&v)[kHeld]) {
            float most = s.m;
#pragma unroll
            for (int q = 0; q < kHeld; ++q) most = fmaxf(most, fmaxf(fmaxf(v[q].x, v[q].y), fmaxf(v[q].z, v[q].w)));
            const float b = base_of(most), d = base_of(s.m) - b;
            s.s0 *= ex(d, a.c0);
            if (TWO) s.s1 *= ex(d, a.c1);
            s.m = most;
#pragma unroll
            for (int q = 0; q < kHeld; ++q) {
                s.s0 += ex(v[q].x - b, a.c0) + ex(v[q].y - b, a.c0) + (ex(v[q].z - b, a.c0) + ex(v[q].w - b, a.c0));
                if (TWO) s.s1 += ex(v[q].x - b, a.c1) + ex(v[q].y - b, a.c1) + (ex(v[q].z - b, a.c1) + ex(v[q].w - b, a.c1));
            }
        };
        unsigned u = part.begin + threadIdx.x;
        for (; u + (kHeld - 1) * THREADS < part.end; u += kHeld * THREADS) {
            float4 v[kHeld];
#pragma unroll
            for (int q = 0; q < kHeld; ++q) v[q] = body[u + q * THREADS];
            take(v);
        }
        if (u < part.end) {
            float4 v[kHeld];
#pragma unroll
            for (int q = 0; q < kHeld; ++q)
                v[q] = u + q * THREADS < part.end ? body[u + q * THREADS] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            take(v);
        }
        s = join_lanes<TWO, 32>(a, s);
        if (lane == 0) of_warp[warp] = s;
    }
    __syncthreads();
    if (GRAD && a.top > kAlone)
        for (unsigned j = threadIdx.x; j < listed; j += THREADS + 32) tokens.insert(j);
    Sums s = join_lanes<TWO, THREADS / 32>(a, of_warp[lane % (THREADS / 32)]);
    if (a.blocks > 1) {
        sm100::cluster_wait();  // the others run: their shared memory is there
        if (warp == 0 && lane < a.blocks) {
            const uint32_t at = sm100::map_to_rank(&of_block[rank], lane);
            sm100::st_cluster(at, s.m);
            sm100::st_cluster(at + 4, s.s0);
            sm100::st_cluster(at + 8, s.s1);
        }
        __syncwarp();
        sm100::cluster_sync_all();
        s = of_block[0];
        for (unsigned r = 1; r < a.blocks; ++r) s = join<TWO>(a, s, of_block[r]);
    }
    const float b = base_of(s.m), s1 = TWO ? s.s1 : s.s0;
    const bool taught = a.soft != 0.f && !(teacher_sum == 0.f);
    const bool labelled = a.hard != 0.f && entries.token[a.top] >= 0;
    if (a.loss && rank == 0 && warp == THREADS / 32) {
        // log p_j - log q_j = (t_j - largest t - (z_j - b)) / T - log sum e + log s0: differences that nearly cancel, in 64 bits
        double total = 0.0, apart = 0.0;
        for (unsigned j = lane; j < a.top; j += 32) {
            const double e = entries.e[j];
            total += e;
            if (e != 0.0) apart += e * (double(entries.t[j]) - (double(entries.z[j]) - double(b)));
        }
        total = sum_of_warp(total);
        apart = sum_of_warp(apart);
        if (lane == 0) {
            double loss = 0.0;
            const double T = a.temperature;
            if (taught) loss += a.soft * (T * T) * (apart / total / T - log(total) + log(double(s.s0)));
            // (the difference first: next to logits of a mask's lowest number the logarithm is nothing)
            if (labelled) loss += a.hard * ((double(b) - double(entries.z[a.top])) + log(double(s1)));
            a.loss[row] = float(weight * loss);
        }
    }
    if (!GRAD) return;
    // ---- the gradient ----
    const float scale = weight * of_row, soft = taught ? scale * a.soft * a.temperature : 0.f, hard = labelled ? scale * a.hard : 0.f;
    const float k0 = TWO ? soft / s.s0 : (soft + hard) / s.s0, k1 = TWO ? hard / s1 : 0.f;
    if (!taught && !labelled) {  // such a row has a loss of 0, whatever it holds
        if (!a.accumulate) zeros();
        return;
    }
    auto slope = [&](float value) {
        const float d = value - b;
        float r = k0 * ex(d, a.c0);
        if (TWO) r += k1 * ex(d, a.c1);
        return r;
    };
    if (warp < THREADS / 32) {
        float4 *out = reinterpret_cast<float4 *>(dz + part.head);
        const bool whole = (reinterpret_cast<uintptr_t>(out) & 15u) == 0;  // the gradient's rows lie as the logits' do
        auto put = [&](unsigned u, float4 v) {
            v = make_float4(slope(v.x), slope(v.y), slope(v.z), slope(v.w));
            if (whole) {
                if (a.accumulate) {
                    const float4 old = out[u];
                    v.x += old.x, v.y += old.y, v.z += old.z, v.w += old.w;
                }
                __stcs(out + u, v);
            } else {
                float *at = dz + part.head + 4 * size_t(u);
                at[0] = a.accumulate ? at[0] + v.x : v.x;
                at[1] = a.accumulate ? at[1] + v.y : v.y;
                at[2] = a.accumulate ? at[2] + v.z : v.z;
                at[3] = a.accumulate ? at[3] + v.w : v.w;
            }
        };
        if (threadIdx.x < part.edge) {
            const unsigned token = part.edge_token(threadIdx.x);
            const float d = slope(z[token]);
            dz[token] = a.accumulate ? dz[token] + d : d;
        }
        unsigned u = part.begin + threadIdx.x;
        for (; u + (kHeld - 1) * THREADS < part.end; u += kHeld * THREADS) {
            float4 v[kHeld];
#pragma unroll
            for (int q = 0; q < kHeld; ++q) v[q] = __ldcs(body + u + q * THREADS);
#pragma unroll
            for (int q = 0; q < kHeld; ++q) put(u + q * THREADS, v[q]);
        }
        if (u < part.end) {
            float4 v[kHeld];
#pragma unroll
            for (int q = 0; q < kHeld; ++q)
                if (u + q * THREADS < part.end) v[q] = __ldcs(body + u + q * THREADS);
#pragma unroll
            for (int q = 0; q < kHeld; ++q)
                if (u + q * THREADS < part.end) put(u + q * THREADS, v[q]);
        }
    }
    __syncthreads();
    if (a.top > kAlone) {
        for (unsigned j = threadIdx.x; j < listed; j += THREADS + 32) tokens.mark(j, entries.e[j]);
        __syncthreads();
    }
    // listed tokens of this block's part, each by its first entry
    for (unsigned j = threadIdx.x; j < listed; j += THREADS + 32) {
        const unsigned token = unsigned(entries.token[j]);
        if (token >= a.vocab || !part.has(token)) continue;
        if (!tokens.is_first(j)) continue;
        float d = 0.f;
        if (taught) d = soft * (tokens.sum(j, entries.e) / teacher_sum);
        if (token == unsigned(entries.token[a.top])) d += hard;
        if (a.accumulate) dz[token] -= d;
        else dz[token] = slope(entries.z[j]) - d;
    }
}

template <int THREADS, bool GRAD, bool TWO>
int32_t launch(katsu_cuda_ctx *ctx, Distill a) {
    const size_t listed = size_t(a.top) + 1;
    a.places = listed_places(listed);
    const size_t array = (listed + 3) / 4 * 4, smem = sizeof(float) * (GRAD ? 5 * array + a.places : 4 * array), blocks = size_t(a.rows) * a.blocks;
    if (blocks > 0x7fffffffu) return katsu_set_error(KATSU_ERR_UNSUPPORTED, "%u rows of %u logits in one loss", a.rows, a.vocab);
    const size_t per_sm = std::min<size_t>(blocks_of_sm(THREADS), katsu_shared_per_sm() / (smem + 2048));
    a.waves = blocks > (a.blocks > 1 ? size_t(ctx->num_sms) * 3 / 4 : per_sm * ctx->num_sms);  // (not every group of SMs is filled by clusters)
    return katsu_launch(ctx, !a.waves, distill_kernel<THREADS, GRAD, TWO>, unsigned(blocks), THREADS + 32, smem, a.blocks, a);
}

template <bool GRAD>
int32_t run(katsu_cuda_ctx *ctx, Distill a) {
    if (a.soft == 0.f || a.top == 0) {  // labels alone: one set of sums, at 1
        a.soft = 0.f;
        a.temperature = 1.f;
        a.top = 0;
    }
    a.c1 = kLog2e;
    a.c0 = kLog2e / a.temperature;
    const bool two = a.hard != 0.f && a.soft != 0.f && a.temperature != 1.f;
    const size_t units = (size_t(a.vocab) + 3) / 4;
    // Threads of a block: few where rows are short and many (8192 rows of 1003: 21.1 us with 128, 14.7 with 64), many where the rows of
    // a gradient are long, as fewer blocks then keep fewer bytes in L2 between their two readings (4096 rows of 32768: 201 us with
    // 256 threads and two blocks a row, 195 with 512 and one).
    const int threads = units <= 1024 && a.rows >= size_t(16) * ctx->num_sms ? 64 : units <= 2048 ? 128 : GRAD && units > 4096 ? 512 : 256;
    a.blocks = 1;
    // Blocks of a row: more where there are few rows; a gradient's, so that all that are resident have their rows in L2.
    while (a.blocks < kMostCluster && units > size_t(a.blocks) * 2 * threads * kHeld &&
           (size_t(a.rows) * a.blocks < size_t(2) * ctx->num_sms || (GRAD && units > a.blocks * size_t(8192))))
        a.blocks *= 2;
    switch (threads) {
        case 64: return two ? launch<64, GRAD, true>(ctx, a) : launch<64, GRAD, false>(ctx, a);
        case 128: return two ? launch<128, GRAD, true>(ctx, a) : launch<128, GRAD, false>(ctx, a);
        case 256: return two ? launch<256, GRAD, true>(ctx, a) : launch<256, GRAD, false>(ctx, a);
        default: return two ? launch<512, true, true>(ctx, a) : launch<512, true, false>(ctx, a);
    }
}

// The checks of both calls.  loss is null where it is not asked for, dlogits in the forward.
int32_t check(const katsu_cuda_ctx *ctx, const Distill &a, size_t rows, size_t vocab, size_t top) {
    KATSU_REQUIRE(ctx != nullptr, "null context");
    KATSU_REQUIRE(rows <= 0x7fffffffu && vocab <= 0x7fffffffu, "rows and vocab are below 2^31");
    KATSU_REQUIRE(top <= KATSU_DISTILL_MAX_TOP, "at most KATSU_DISTILL_MAX_TOP entries of a row");
    KATSU_REQUIRE(a.temperature >= FLT_MIN && isfinite(a.temperature), "temperature must be above 0, and finite");  // (its reciprocal too)
    KATSU_REQUIRE(isfinite(a.soft) && isfinite(a.hard), "soft and hard must be finite");
    if (rows == 0) return KATSU_OK;
    KATSU_REQUIRE(vocab != 0, "a loss needs a vocabulary");
    KATSU_REQUIRE(a.logits != nullptr, "logits is null");
    KATSU_REQUIRE(top == 0 || a.soft == 0.f || (a.teacher != nullptr && a.index != nullptr), "teacher or index is null");
    const struct {
        const void *p;
        size_t bytes;
    } in[] = {{a.logits, 4 * rows * vocab}, {a.teacher, 4 * rows * top}, {a.index, 4 * rows * top}, {a.labels, 4 * rows}, {a.weight, 4 * rows},
              {a.g, 4 * rows}}, out[] = {{a.dlogits, 4 * rows * vocab}, {a.loss, 4 * rows}};
    for (const auto &o : out) {
        KATSU_REQUIRE(katsu_whole(o.p), "an address is not that of a whole element");
        for (const auto &i : in) {
            // the logits' place: of the gradient and these two operands alone, whatever else is at their address
            const bool in_place = &o == out && &i == in && o.p == i.p && !a.accumulate;
            KATSU_REQUIRE(katsu_whole(i.p), "an address is not that of a whole element");
            KATSU_REQUIRE(in_place || !katsu_overlap(o.p, o.bytes, i.p, i.bytes), "an output is an input too, or overlaps one");
        }
    }
    KATSU_REQUIRE(!katsu_overlap(out[0].p, out[0].bytes, out[1].p, out[1].bytes), "loss and dlogits overlap");
    return KATSU_OK;
}

}  // namespace

extern "C" int32_t katsu_cuda_distill_fwd(katsu_cuda_ctx *ctx, const float *logits, const float *teacher, const int32_t *index,
                                          const int32_t *labels, const float *weight, float temperature, float soft, float hard,
                                          float *loss, size_t rows, size_t vocab, size_t top) {
    const Distill a = {logits, teacher, weight, nullptr, index, labels, loss, nullptr, temperature, soft, hard,
                       0.f, 0.f, unsigned(rows), unsigned(vocab), unsigned(top), 1, 0, 0, 0};
    KATSU_TRY(check(ctx, a, rows, vocab, top));
    KATSU_REQUIRE(loss != nullptr || rows == 0, "loss is null");
    KATSU_TRY(katsu_bind(ctx));
    return rows ? run<false>(ctx, a) : KATSU_OK;
}

extern "C" int32_t katsu_cuda_distill_bwd(katsu_cuda_ctx *ctx, const float *logits, const float *teacher, const int32_t *index,
                                          const int32_t *labels, const float *weight, float temperature, float soft, float hard,
                                          const float *g, float *loss, float *dlogits, size_t rows, size_t vocab, size_t top,
                                          int32_t accumulate) {
    const Distill a = {logits, teacher, weight, g, index, labels, loss, dlogits, temperature, soft, hard,
                       0.f, 0.f, unsigned(rows), unsigned(vocab), unsigned(top), 1, 0, accumulate != 0, 0};
    KATSU_TRY(check(ctx, a, rows, vocab, top));
    KATSU_REQUIRE(dlogits != nullptr || rows == 0, "dlogits is null");
    KATSU_TRY(katsu_bind(ctx));
    return rows ? run<true>(ctx, a) : KATSU_OK;
}
