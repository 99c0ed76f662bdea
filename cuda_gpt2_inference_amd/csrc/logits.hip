// logits.hip -- rules on logits, and their probabilities, on MI355X (gfx950): penalties for tokens that a sequence
// holds, biases, grammar masks, then the logits or softmax(x / temperature).
//
//   x   = logit; of a token that the sequence holds x / r where positive, else x r      (repetition r)
//   x  -= frequency * count + (count > 0 ? presence : 0)                               (count: times generated)
//   x  += bias;   x = -inf where the grammar forbids the token
//
// A row is read once, stays in registers between the maximum, the sum and the quotient, and is written once.  What a
// sequence holds is a list of ids, so the tokens that any rule names are few against the vocabulary: they are set bits of
// a map in LDS (a bit a token), and a token's place among the set bits, from a prefix sum over the map's words, is its
// entry in a table: a thread for every entry works its logit out.  A row's four neighbouring tokens look at four
// bits, and only where one is set at the table.  In slices of a row whose counts fit beside another workgroup's, the table
// has an entry for every token (counts, that each thread works its own logits out from), which takes no map, no places and
// fewer barriers.  The row of a token of a tree holds its branch too (the bits of its mask), so every row builds its own table.
// (Eight rows of a sequence in one workgroup with one table: 32 trees of up to 8 rows 24 us in place of 19, since fewer
// workgroups hide the same chain of loads and barriers.)
//
// A row on one CU takes the CU's time for its arithmetic (a dozen instructions a token and the table: 19 us for one row of
// 50257), so few rows are cut into slices, a workgroup each (7 us).  Of probabilities the slices of a row exchange their
// maxima and sums as tagged words in the workspace, while all of them are on the GPU; a slice that waits in vain works the
// missing ones out itself.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>

#include "lanes.hpp"
#include "tree.hpp"

namespace {

constexpr int kRun = 4;                        // neighbouring tokens of a thread
constexpr int kSliceThreads = 512, kRowThreads = 1024;     // of a slice's workgroup, of a whole row's
constexpr int kMostSlices = 64;                // of a row whose slices exchange words: a lane each
constexpr int kTogether = 512;                 // workgroups of kSliceThreads that run at once: two a CU
constexpr int kMaxVocab = 1 << 18;
constexpr int kMaxRows = 1 << 21;              // whole rows of a grid: 2^32 threads are too many
constexpr int kMaxSequences = 1 << 20;
constexpr int kSmallRuns = 2;                  // of a slice of logits whose table has biases too
constexpr int kIds = 8, kNamed = 2;             // ids and named tokens of a thread that are asked for ahead
constexpr int kLdsMost = 156 * 1024;           // a CU's, less what is static here
constexpr int kLdsTogether = 76 * 1024;        // two workgroups a CU
constexpr float kLog2e = 1.4426950408889634f;

struct LogitArgs {
    void* out;
    const void* x;
    const int* start;
    kvattn_logit_rules r;
    size_t in_row, out_row;
    int B, rows, V, words, entries;            // words of the map; entries of the table
    int row0;                                  // the launch's first row
    int slices, slice;                         // of a row, tokens of one
    unsigned long long* exchange;              // [rows of the launch][slices][2] tagged words
    int polls;
    bool vec;                                  // rows start on boundaries of a run
};

template <bool kF32>
__device__ __forceinline__ float logit(const void* p, size_t i) {
    if constexpr (kF32) return reinterpret_cast<const float*>(p)[i];
    else return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}

// vec: rows start on boundaries of a run.
template <bool kF32>
__device__ __forceinline__ void load_run(const void* p, size_t row0, int v, int V, bool vec, float (&x)[kRun]) {
    if (vec && v + kRun <= V) {
        if constexpr (kF32) {
            const float4 w = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + row0 + v);
            x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + row0 + v);
            x[0] = bf16_lo(w.x); x[1] = bf16_hi(w.x); x[2] = bf16_lo(w.y); x[3] = bf16_hi(w.y);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i) x[i] = v + i < V ? logit<kF32>(p, row0 + min(v + i, V - 1)) : -INFINITY;
}

template <bool kF32>
__device__ __forceinline__ void store_run(void* p, size_t row0, int v, int V, bool vec, const float (&x)[kRun]) {
    if (vec && v + kRun <= V) {
        if constexpr (kF32) {
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + row0 + v) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + row0 + v) =
                make_uint2(f32_to_bf16(x[0]) | (uint32_t)f32_to_bf16(x[1]) << 16, f32_to_bf16(x[2]) | (uint32_t)f32_to_bf16(x[3]) << 16);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        if (v + i >= V) return;
        if constexpr (kF32) reinterpret_cast<float*>(p)[row0 + v + i] = x[i];
        else reinterpret_cast<uint16_t*>(p)[row0 + v + i] = f32_to_bf16(x[i]);
    }
}

// The last of B sequences that begins at or before the row, 64 looked at at once.
__device__ __forceinline__ int sequence_of(const int* start, int B, int row, int lane) {
    int b = 0;
    for (int step = B > kWave * kWave * kWave ? kWave * kWave * kWave : B > kWave * kWave ? kWave * kWave : B > kWave ? kWave : 1;; step /= kWave) {
        const int i = b + lane * step;
        const unsigned long long at = __ballot(i < B && start[min(i, B - 1)] <= row);
        b += (63 - __clzll((long long)(at | 1))) * step;
        if (step == 1) break;
    }
    return b;
}

// kRuns: runs of a thread that are kept in registers; 0: of a longer row none is, and each pass reads it again.
// kShare: the row's probabilities are those of several workgroups.
// kDense: the table has an entry for every token, which spares the places, their barriers and gathered logits.
template <bool kInF32, bool kOutF32, bool kProbs, int kThreads, int kRuns, bool kShare, bool kDense>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4))) void logits_kernel(LogitArgs a) {
    constexpr int kWaves = kThreads / kWave, kStep = kThreads * kRun;      // tokens from one run of a thread to its next
    static_assert(!kShare || (kProbs && kRuns > 0), "slices in registers");
    extern __shared__ __align__(16) uint32_t lds[];    // map, allowed tokens, named tokens, counts, biases, prefixes (16 bits)
    __shared__ uint32_t wave_words[kWaves];
    __shared__ float wave_floats[2][kWaves];
    __shared__ unsigned long long wave_keys[kWaves];
    __shared__ float slice_top[kMostSlices], slice_sum[kMostSlices];       // (sum: of the likeliest token alone, its number)
    __shared__ unsigned long long missing_at;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int launch_row = a.slices > 1 ? blockIdx.x / a.slices : blockIdx.x, row = a.row0 + launch_row;
    const int own = a.slices > 1 ? blockIdx.x - launch_row * a.slices : 0;
    constexpr int kHeld = kRuns ? kRuns : 1;
    float x[kHeld][kRun];
    const size_t in0 = (size_t)row * a.in_row, out0 = (size_t)row * a.out_row;
    int v0 = own * a.slice, v1 = min(a.V, v0 + a.slice);      // this workgroup's tokens
    auto load = [&] {
        if constexpr (kRuns > 0) {
#pragma unroll
            for (int j = 0; j < kRuns; ++j) load_run<kInF32>(a.x, in0, v0 + tid * kRun + j * kStep, v1, a.vec, x[j]);
        }
    };
    // Loads come back in order: those that others depend on are asked for before the row.
    int first = 0, end = 0;
    if (a.start) {
        first = a.start[min(lane, a.B - 1)];
        end = a.start[a.B];
    }
    asm volatile("" ::: "memory");
    load();
    asm volatile("" ::: "memory");
    int b = row, t0 = row;
    if (a.start) {
        if (row >= end) return;                // behind the last token
        b = a.B <= kWave ? 63 - __clzll((long long)(__ballot(lane < a.B && first <= row) | 1)) : sequence_of(a.start, a.B, row, lane);
        t0 = min(max(a.start[b], 0), row);
    }

    // What the sequence holds is asked for before its length is known (places behind it are not looked at).
    const bool table = a.entries > 0;
    const int* const history = a.r.history + (size_t)b * a.r.max_history;
    int ids[kIds];
    if (a.r.history) {
#pragma unroll
        for (int k = 0; k < kIds; ++k) ids[k] = k * kThreads < a.r.max_history ? history[min(tid + k * kThreads, a.r.max_history - 1)] : -1;
    }
    const float temperature = a.r.temperature ? a.r.temperature[b] : 1.0f;
    // (Of a dense table counts, biases and allowed tokens alone.)
    uint32_t* const map = lds;
    uint32_t* const names = map + a.words;
    uint32_t* const count = kDense ? lds : names + a.entries;
    uint32_t* const bias_at = count + (kDense && !table ? 0 : a.entries);
    uint32_t* const allowed = bias_at + (a.r.bias_start ? a.entries : 0);
    uint16_t* const before = reinterpret_cast<uint16_t*>(allowed + (a.r.allowed ? a.words : 0));
    int line = -1;
    if (a.r.allowed) line = a.r.allowed_of ? a.r.allowed_of[row] : row;
    const bool grammar = a.r.allowed && line >= 0 && line < a.r.num_allowed;

    int held = 0, prompt = 0, branch = -1, bias0 = 0, biases = 0, bias_id = -1;
    float repetition = 1.0f, frequency = 0.0f, presence = 0.0f;
    if (table) {
        held = a.r.history ? min(max(a.r.history_len[b], 0), a.r.max_history) : 0;
        prompt = a.r.prompt_len ? a.r.prompt_len[b] : 0;
        if (a.r.repetition) repetition = a.r.repetition[b];
        if (a.r.frequency) frequency = a.r.frequency[b];
        if (a.r.presence) presence = a.r.presence[b];
        // This thread's token of the row's branch, and the sequence's biases.
        if (a.r.tokens && tid < 64 * a.r.mask_words) {
            // (Bits behind the sequence's last row are no tokens of it.)
            const int its = a.r.tokens[min(t0 + tid, a.rows - 1)], last = min(a.start ? a.start[b + 1] : row + 1, a.rows);
            if (t0 + tid < last && (a.r.masks[(size_t)row * a.r.mask_words + (tid >> 6)] >> (tid & 63)) & 1) branch = its;
        }
        if (a.r.bias_start) {
            bias0 = min(max(a.r.bias_start[b], 0), a.r.num_bias);
            biases = min(min(max(a.r.bias_start[b + 1], bias0), a.r.num_bias) - bias0, a.r.max_bias);
            if (tid < biases) bias_id = a.r.bias_ids[bias0 + tid];
        }
    }
    auto each_bias = [&](auto&& f) {
        if (tid < biases) f(bias_id, bias0 + tid);
        for (int i = tid + kThreads; i < biases; i += kThreads) f(a.r.bias_ids[bias0 + i], bias0 + i);
    };
    // A held or biased token's logit.
    auto adjusted = [&](float z, uint32_t c, uint32_t from) {
#pragma clang fp contract(off)
        const float made = (float)((c & 0xffffu) - (c >> 16));
        if (c) z = z > 0.0f ? z / repetition : z * repetition;
        z = z - (frequency * made + (made > 0.0f ? presence : 0.0f));
        if (from) z = z + a.r.bias[from - 1];
        return z;
    };
    // Allowed and named tokens of v0 .. v1 - 1.
    auto build = [&] {
        const int first = v0 >> 5, words = (v1 - v0 + 31) >> 5;
        if (grammar)
            for (int w = tid; w < words; w += kThreads) allowed[w] = a.r.allowed[(size_t)line * a.r.allowed_stride + first + w];
        if (!table) return;
        auto known = [&](int id) { return id >= v0 && id < v1; };
        auto each_held = [&](auto&& f) {
#pragma unroll
            for (int k = 0; k < kIds; ++k)
                if (tid + k * kThreads < held) f(ids[k], tid + k * kThreads);
            for (int i = tid + kIds * kThreads; i < held; i += kThreads) f(history[i], i);
        };
        if constexpr (kDense) {
            const int all = (a.r.bias_start ? 2 : 1) * a.entries;          // (a multiple of 4)
            for (int e = 4 * tid; e < all; e += 4 * kThreads) *reinterpret_cast<uint4*>(count + e) = make_uint4(0, 0, 0, 0);
            __syncthreads();
            // Times held in the lower half, times of those in the prompt in the upper: at most 2^15 each.
            each_held([&](int id, int i) {
                if (known(id)) atomicAdd(count + (id - v0), i < prompt ? 0x10001u : 1u);
            });
            if (known(branch)) atomicAdd(count + (branch - v0), 1u);
            each_bias([&](int id, int i) {     // of an id listed twice the last
                if (known(id)) atomicMax(bias_at + (id - v0), (uint32_t)(i + 1));
            });
            return;
        }
        for (int w = tid; w < words; w += kThreads) map[w] = 0;
        __syncthreads();
        auto mark = [&](int id) {              // (text repeats itself: mostly it is marked)
            if (known(id) && !((map[(id - v0) >> 5] >> (id & 31)) & 1)) atomicOr(map + ((id - v0) >> 5), 1u << (id & 31));
        };
        each_held([&](int id, int) { mark(id); });
        mark(branch);
        each_bias([&](int id, int) { mark(id); });
        __syncthreads();
        // Set bits before every word: a thread's words, then the threads'.
        const int per = (words + kThreads - 1) / kThreads, w0 = min(tid * per, words), w1 = min(w0 + per, words);
        uint32_t mine = 0;
        for (int w = w0; w < w1; ++w) mine += __popc(map[w]);
        uint32_t upto = mine;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const uint32_t o = __shfl_up(upto, d);
            if (lane >= d) upto += o;
        }
        if (lane == kWave - 1) wave_words[wave] = upto;
        __syncthreads();
        uint32_t at = upto - mine, all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) at += wave_words[w];
            all += wave_words[w];
        }
        for (int w = w0; w < w1; ++w) {
            before[w] = (uint16_t)at;
            for (uint32_t bits = map[w]; bits; bits &= bits - 1) names[at++] = v0 + 32 * w + __builtin_ctz(bits);
        }
        for (uint32_t e = tid; e < all; e += kThreads) {
            count[e] = 0;
            if (a.r.bias_start) bias_at[e] = 0;
        }
        __syncthreads();
        // The named tokens' logits are asked for while they are counted.
        float named[kNamed];
#pragma unroll
        for (int k = 0; k < kNamed; ++k) named[k] = tid + k * kThreads < all ? logit<kInF32>(a.x, in0 + names[tid + k * kThreads]) : 0.0f;
        auto entry = [&](int id) { return before[(id - v0) >> 5] + __popc(map[(id - v0) >> 5] & ((1u << (id & 31)) - 1)); };
        each_held([&](int id, int i) {
            if (known(id)) atomicAdd(count + entry(id), i < prompt ? 0x10001u : 1u);
        });
        if (known(branch)) atomicAdd(count + entry(branch), 1u);
        each_bias([&](int id, int i) {
            if (known(id)) atomicMax(bias_at + entry(id), (uint32_t)(i + 1));
        });
        __syncthreads();
        // A thread for every named token: its logit takes its count's place.
        auto adjust = [&](uint32_t e, float z) {
            count[e] = __float_as_uint(adjusted(z, count[e], a.r.bias_start ? bias_at[e] : 0));
        };
#pragma unroll
        for (int k = 0; k < kNamed; ++k)
            if (tid + k * kThreads < all) adjust(tid + k * kThreads, named[k]);
        for (uint32_t e = tid + kNamed * kThreads; e < all; e += kThreads) adjust(e, logit<kInF32>(a.x, in0 + names[e]));
    };
    auto rules = [&](int v, float (&y)[kRun]) {
        if (v >= v1) return;
        const int w = (v - v0) >> 5;
        if (kDense && table) {
            const uint4 c = *reinterpret_cast<const uint4*>(count + (v - v0));
            const uint4 f = a.r.bias_start ? *reinterpret_cast<const uint4*>(bias_at + (v - v0)) : make_uint4(0, 0, 0, 0);
            if (c.x | c.y | c.z | c.w | f.x | f.y | f.z | f.w) {
                const uint32_t cs[kRun] = {c.x, c.y, c.z, c.w}, fs[kRun] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int i = 0; i < kRun; ++i)
                    if (cs[i] | fs[i]) y[i] = adjusted(y[i], cs[i], fs[i]);
            }
        } else if (table) {
            const uint32_t word = map[w], bits = (word >> (v & 31)) & 15u;
            if (bits) {
                // (Entries of the run are neighbours; those before its first bit and behind its last are read for nothing.)
                uint32_t e = before[w] + __popc(word & ((1u << (v & 31)) - 1));
                uint32_t z[kRun];
#pragma unroll
                for (int i = 0; i < kRun; ++i) {
                    z[i] = count[e];
                    if (i + 1 < kRun) e = min(e + ((bits >> i) & 1), (uint32_t)a.entries - 1);
                }
#pragma unroll
                for (int i = 0; i < kRun; ++i) y[i] = (bits >> i) & 1 ? __uint_as_float(z[i]) : y[i];
            }
        }
        if (grammar) {
            const uint32_t ok = allowed[w] >> (v & 31);
#pragma unroll
            for (int i = 0; i < kRun; ++i) y[i] = (ok >> i) & 1 ? y[i] : -INFINITY;
        }
    };
    // Every run of the thread, with the rules applied.
    auto each = [&](auto&& f) {
        if constexpr (kRuns > 0) {
#pragma unroll
            for (int j = 0; j < kRuns; ++j) f(v0 + tid * kRun + j * kStep, x[j]);
        } else {
            for (int v = v0 + tid * kRun; v < v1; v += kStep) {
                load_run<kInF32>(a.x, in0, v, v1, a.vec, x[0]);
                rules(v, x[0]);
                f(v, x[0]);
            }
        }
    };
    auto apply = [&] {
        build();
        if (table || a.r.allowed) __syncthreads();
        if constexpr (kRuns > 0) {
#pragma unroll
            for (int j = 0; j < kRuns; ++j) rules(v0 + tid * kRun + j * kStep, x[j]);
        }
    };
    apply();
    if constexpr (!kProbs) {
        each([&](int v, float (&y)[kRun]) { store_run<kOutF32>(a.out, out0, v, v1, a.vec, y); });
        return;
    }
    const bool likeliest = !(temperature > 0.0f);
    // (A factor of zero or infinity would make NaN of forbidden tokens, and of the likeliest.)
    const float scale = fminf(fmaxf(kLog2e / temperature, FLT_MIN), FLT_MAX);
    float top = -INFINITY, sum = 0.0f;         // of this workgroup's tokens
    int token = -1;                            // its likeliest, the lowest of several
    auto weigh = [&](float (&y)[kRun]) {
#pragma unroll
        for (int i = 0; i < kRun; ++i) y[i] = exp2_fast((y[i] - top) * scale);
    };
    // The tokens' maximum, and the sum of their weights against it (in their places), or which one is the largest.
    auto reduce = [&] {
        top = -INFINITY;
        each([&](int, float (&y)[kRun]) {
#pragma unroll
            for (int i = 0; i < kRun; ++i) top = fmaxf(top, y[i]);
        });
        top = wave_max(top);
        if (lane == 0) wave_floats[0][wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_floats[0][w]);
        if (likeliest || top == -INFINITY) {
            unsigned long long best = 0;
            each([&](int v, float (&y)[kRun]) {
#pragma unroll
                for (int i = 0; i < kRun; ++i) {
                    const unsigned long long key = 0xffffffffu - (uint32_t)(v + i);
                    if (y[i] == top && v + i < v1 && key > best) best = key;
                }
            });
#pragma unroll
            for (int d = 1; d < kWave; d *= 2) {
                const unsigned long long o = __shfl_xor(best, d);
                best = o > best ? o : best;
            }
            if (lane == 0) wave_keys[wave] = best;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaves; ++w) best = wave_keys[w] > best ? wave_keys[w] : best;
            token = top == -INFINITY ? -1 : (int)(0xffffffffu - (uint32_t)best);
            sum = 0.0f;
            // NaN, which maxima pass over, makes the sum NaN beside a number; without one it is found here, as every sum of
            // -inf alone is -inf.  (Weights taken against zero would show it too, but beside that branch alone the compiler
            // spills a hundred registers of 13 runs: 256 rows 43 us in place of 31.)
            if (!likeliest) {
                each([&](int, float (&y)[kRun]) { sum += (y[0] + y[1]) + (y[2] + y[3]); });
                sum = wave_sum(sum);
                if (lane == 0) wave_floats[1][wave] = sum;
                __syncthreads();
                sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) sum += wave_floats[1][w];
                sum = sum == sum ? 0.0f : sum;
            }
        } else {
            sum = 0.0f;
            each([&](int, float (&y)[kRun]) {
                weigh(y);
                sum += (y[0] + y[1]) + (y[2] + y[3]);
            });
            sum = wave_sum(sum);
            if (lane == 0) wave_floats[1][wave] = sum;
            __syncthreads();
            sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) sum += wave_floats[1][w];
        }
    };
    reduce();
    float one = 1.0f / sum;                    // what a weight is multiplied with
    bool none = top == -INFINITY && sum == 0.0f;
    if constexpr (kShare) {
        // A slice's words: its maximum; its sum, or its likeliest token.
        unsigned long long* const words = a.exchange + (size_t)launch_row * a.slices * 2;
        const uint32_t tag = call_tag();
        if (tid == 0) {
            publish_word(words + 2 * own, tagged_word(top, tag), false);
            publish_word(words + 2 * own + 1, tagged_word(likeliest ? __int_as_float(token) : sum, tag), false);
        }
        if (wave == 0) {
            unsigned long long w0 = 0, w1 = 0;
            bool ok = false;
            for (int r = 0; r < a.polls; ++r) {
                if (!ok) {
                    w0 = get_word(words + 2 * min(lane, a.slices - 1));
                    w1 = get_word(words + 2 * min(lane, a.slices - 1) + 1);
                    ok = word_is(w0, tag) && word_is(w1, tag);
                }
                if (__all(ok)) break;
            }
            if (lane == own) {                 // (also where nothing was waited for)
                ok = true;
                w0 = tagged_word(top, tag);
                w1 = tagged_word(likeliest ? __int_as_float(token) : sum, tag);
            }
            slice_top[lane] = word_value(w0);
            slice_sum[lane] = word_value(w1);
            const unsigned long long out = __ballot(!ok && lane < a.slices);
            if (lane == 0) missing_at = out;
        }
        __syncthreads();
        // Slices that have not come are worked out here, then this one again.
        unsigned long long missing = missing_at;
        if (missing) {
            missing |= 1ull << own;
            const int order_own = own;
            while (missing) {
                const unsigned long long others = missing & ~(1ull << order_own);
                const int s = others ? __ffsll((long long)others) - 1 : order_own;
                missing &= ~(1ull << s);
                v0 = s * a.slice;
                v1 = min(a.V, v0 + a.slice);
                __syncthreads();
                load();
                apply();
                reduce();
                if (tid == 0) {
                    slice_top[s] = top;
                    slice_sum[s] = likeliest ? __int_as_float(token) : sum;
                }
                __syncthreads();
            }
        }
        // A lane for every slice.
        const float its_top = lane < a.slices ? slice_top[lane] : -INFINITY, its_sum = lane < a.slices ? slice_sum[lane] : 0.0f;
        const float all = wave_max(its_top);
        none = all == -INFINITY;
        if (likeliest) {
            const unsigned long long at = __ballot(its_top == all);
            token = __builtin_amdgcn_readlane(__float_as_int(its_sum), __ffsll((long long)(at | 1ull << 63)) - 1);
        } else {
            // (A slice without a number has a sum of zero, or NaN, and its maximum may not be taken a difference of.)
            const float total = wave_sum(its_top == -INFINITY ? its_sum : exp2_fast((its_top - all) * scale) * its_sum);
            none = none && total == 0.0f;
            // (Beside an infinity in another slice nothing weighs anything.)
            const float part = top == -INFINITY ? 0.0f : exp2_fast((top - all) * scale);
            one = part == 0.0f ? 0.0f : part / total;
        }
    }
    if (likeliest || none || top == -INFINITY) {
        // The likeliest token alone; nothing where no token is left; of tokens without a number among them, whose logits were
        // left as they are, NaN alone.
        each([&](int v, float (&y)[kRun]) {
#pragma unroll
            for (int i = 0; i < kRun; ++i) {
                const float other = likeliest || none || y[i] == y[i] ? 0.0f : y[i];
                y[i] = likeliest && !none && v + i == token ? 1.0f : other;
            }
            store_run<kOutF32>(a.out, out0, v, v1, a.vec, y);
        });
        return;
    }
    each([&](int v, float (&y)[kRun]) {
        if constexpr (kRuns == 0) weigh(y);
        // (A forbidden token has none, also where the others' is NaN.)
#pragma unroll
        for (int i = 0; i < kRun; ++i) y[i] = y[i] == 0.0f ? 0.0f : y[i] * one;
        store_run<kOutF32>(a.out, out0, v, v1, a.vec, y);
    });
}

// How a call runs: threads and runs of a workgroup, its slices of a row.
struct LogitPlan {
    const void* fn;
    int threads, tokens, slices;               // tokens of a slice
    bool dense;                                // its table has an entry for every token
};
template <bool kInF32, bool kOutF32, bool kProbs, int kRuns, bool kDense>
LogitPlan slices_plan(int V) {
    const int tokens = kSliceThreads * kRun * kRuns, slices = (V + tokens - 1) / tokens;
    const void* fn = (const void*)&logits_kernel<kInF32, kOutF32, kProbs, kSliceThreads, kRuns, false, kDense>;
    if constexpr (kProbs) {
        if (slices > 1) fn = (const void*)&logits_kernel<kInF32, kOutF32, kProbs, kSliceThreads, kRuns, true, kDense>;
    }
    return {fn, kSliceThreads, tokens, slices, kDense};
}
template <bool kInF32, bool kOutF32, bool kProbs>
LogitPlan plan_for(int rows, int V, bool share, const kvattn_logit_rules& r) {
    // The smallest slices with which a call's workgroups run at once; of logits alone, which wait for none, up to 8192
    // tokens.  us per call, 50257 logits:
    //   probabilities of 1 row, history of 1000: slices 6.9, one workgroup 19.4; 64: 12.1 / 21.4; 256: 30.7 / 31.0
    //   64 rows, slices of 8192, an entry for every token or for the named: history of 10 10.5 / 11.7, 2000 12.6 / 13.9, 100 and
    //     biases 11.7 / 12.4, 8000 and biases 16.2 / 32.4; 120 rows, of 16384, history of 10 17.6 / 18.3, 5000 24.0 / 24.8, 20000
    //     32.6 / 79.4 (with biases the entries do not fit beside another workgroup's)
    //   logits of 2000 rows, history of 2000, slices of 8192 tokens, 4096, 16384: 184, 225, 258; of 250 rows 24.2, 28.0, 31.6;
    //     of 144 rows with biases, history of 4000: 23.9, 21.3, 42.4
    constexpr int kToken = kSliceThreads * kRun;
    auto fits = [&](int runs) {
        const long long slices = (V + kToken * runs - 1) / (kToken * runs);
        if (!kProbs) return rows * slices <= kTogether + kTogether / 4;
        return slices == 1 || (share && slices <= kMostSlices && rows * slices <= kTogether);
    };
    if (fits(1)) return slices_plan<kInF32, kOutF32, kProbs, 1, true>(V);
    if (fits(kSmallRuns) || (!kProbs && r.bias_start)) return slices_plan<kInF32, kOutF32, kProbs, kSmallRuns, true>(V);
    if (!kProbs || fits(4)) return slices_plan<kInF32, kOutF32, kProbs, 4, true>(V);
    if constexpr (kProbs) {
        if (fits(8) && !r.bias_start) return slices_plan<kInF32, kOutF32, kProbs, 8, true>(V);
        if (fits(8)) return slices_plan<kInF32, kOutF32, kProbs, 8, false>(V);
        if (fits(13)) return slices_plan<kInF32, kOutF32, kProbs, 13, false>(V);
        constexpr int kRowToken = kRowThreads * kRun;
        if (V <= 13 * kRowToken) return {(const void*)&logits_kernel<kInF32, kOutF32, true, kRowThreads, 13, false, false>, kRowThreads, V, 1, false};
    }
    return {(const void*)&logits_kernel<kInF32, kOutF32, true, kRowThreads, 0, false, false>, kRowThreads, V, 1, false};
}
template <bool kInF32>
LogitPlan plan_for(int rows, int V, bool out_f32, bool probs, bool share, const kvattn_logit_rules& r) {
    if (out_f32) return probs ? plan_for<kInF32, true, true>(rows, V, share, r) : plan_for<kInF32, true, false>(rows, V, share, r);
    return probs ? plan_for<kInF32, false, true>(rows, V, share, r) : plan_for<kInF32, false, false>(rows, V, share, r);
}

int hip_status(hipError_t e) {
    if (e == hipSuccess) return KVATTN_OK;
    kvattn_internal::set_last_hip_error((int)e);
    return KVATTN_ERR_HIP;
}

}  // namespace

extern "C" size_t kvattn_logits_workspace_bytes(void) { return (size_t)kTogether * 2 * sizeof(unsigned long long); }

extern "C" int kvattn_process_logits(void* out, const void* logits, const kvattn_logit_rules* rules,
                                     const int* token_start, int B, int rows, int V, long long row_stride,
                                     long long out_stride, int dtype, int out_dtype, int probs, void* stream) {
    if ((dtype != KVATTN_KV_F32 && dtype != KVATTN_KV_BF16) || (out_dtype != KVATTN_KV_F32 && out_dtype != KVATTN_KV_BF16))
        return KVATTN_ERR_DTYPE;
    if (B < 1 || B > kMaxSequences || rows < 0 || rows > kMaxRows || V < 1 || V > kMaxVocab || row_stride < V || out_stride < V)
        return KVATTN_ERR_SHAPE;
    if (!token_start && rows != B) return KVATTN_ERR_SHAPE;
    LogitArgs a{};
    if (rules) a.r = *rules;
    kvattn_logit_rules& r = a.r;
    const bool branches = r.tokens || r.masks;
    if ((r.history && (r.max_history < 1 || r.max_history > (1 << 15))) || (branches && (r.mask_words < 1 || r.mask_words > kvattn_internal::kMaxMaskWords)) ||
        (r.bias_start && (r.num_bias < 0 || r.max_bias < 0 || r.max_bias > (1 << 15))) ||
        (r.allowed && (r.num_allowed < 1 || r.allowed_stride < (V + 31) / 32)))
        return KVATTN_ERR_SHAPE;
    if (rows == 0) return KVATTN_OK;
    if (!out || !logits || (r.history && !r.history_len) || (branches && (!r.tokens || !r.masks)) ||
        (r.bias_start && r.num_bias > 0 && (!r.bias_ids || !r.bias)))
        return KVATTN_ERR_NULL_POINTER;
    const size_t in = dtype == KVATTN_KV_F32 ? 4 : 2, res = out_dtype == KVATTN_KV_F32 ? 4 : 2;
    const void* words[] = {token_start, r.history, r.history_len, r.prompt_len, r.tokens, r.repetition, r.frequency, r.presence,
                           r.temperature, r.bias_start, r.bias_ids, r.bias, r.allowed, r.allowed_of};
    for (const void* p : words)
        if ((uintptr_t)p & 3u) return KVATTN_ERR_MISALIGNED;
    if (r.workspace && r.workspace_bytes < kvattn_logits_workspace_bytes()) return KVATTN_ERR_WORKSPACE;
    if (((uintptr_t)r.workspace & 7u) || ((uintptr_t)r.masks & 7u) || ((uintptr_t)logits % in) || ((uintptr_t)out % res)) return KVATTN_ERR_MISALIGNED;
    if (r.bias_start && (r.num_bias == 0 || r.max_bias == 0)) r.bias_start = nullptr;
    a.out = out;
    a.x = logits;
    a.start = token_start;
    a.in_row = (size_t)row_stride;
    a.out_row = (size_t)out_stride;
    a.B = B;
    a.rows = rows;
    a.V = V;
    // Every entry is another token: a workgroup has no more of them than of these.
    const int named = (r.history ? r.max_history : 0) + (branches ? 64 * r.mask_words : 0) + (r.bias_start ? r.max_bias : 0);
    const auto lds_of = [&](const LogitPlan& p) {
        a.words = (std::min(V, p.tokens) + 31) / 32;
        a.entries = named == 0 ? 0 : p.dense ? p.tokens : std::min(std::min(V, p.tokens), named);
        const size_t masks = r.allowed ? (size_t)a.words * 4 : 0, entry = p.dense ? 4 : 8;
        return masks + (size_t)a.entries * (entry + (r.bias_start ? 4 : 0)) + (p.dense ? 0 : (size_t)a.words * 4 + (size_t)(a.words + 1) / 2 * 4);
    };
    a.vec = row_stride % kRun == 0 && out_stride % kRun == 0 && ((uintptr_t)logits % (kRun * in)) == 0 &&
            ((uintptr_t)out % (kRun * res)) == 0;
    const bool out_f32 = out_dtype == KVATTN_KV_F32;
    const auto plan = [&](int n, bool share) {
        return dtype == KVATTN_KV_F32 ? plan_for<true>(n, V, out_f32, probs != 0, share, r)
                                       : plan_for<false>(n, V, out_f32, probs != 0, share, r);
    };
    // Slices may have to read one another's logits again, which must still be there.
    const uintptr_t x0 = (uintptr_t)logits, y0 = (uintptr_t)out;
    const uintptr_t x1 = x0 + ((size_t)(rows - 1) * row_stride + V) * in, y1 = y0 + ((size_t)(rows - 1) * out_stride + V) * res;
    const bool share = r.workspace && (y1 <= x0 || x1 <= y0);
    LogitPlan p = plan(rows, share);
    size_t lds = lds_of(p);
    int launch_rows = rows;
    if (probs && share && lds > (p.slices > 1 ? kLdsTogether : kLdsMost)) {
        // Long tables, of slices that would not run at once, or of rows: some rows at a time, in slices whose tables have an
        // entry for every token.
        const int slices = (V + 4 * kSliceThreads * kRun - 1) / (4 * kSliceThreads * kRun);
        launch_rows = std::max(1, kTogether / slices);
        p = plan(launch_rows, true);
        lds = lds_of(p);
    }
    if (lds > kLdsMost) return KVATTN_ERR_LDS;
    // (Nor may a grid of slices have 2^32 threads.)
    launch_rows = (int)std::min<long long>(launch_rows, ((1ll << 32) - 1) / ((long long)p.slices * p.threads));
    a.slices = p.slices;
    a.slice = p.tokens;
    a.exchange = (unsigned long long*)r.workspace;
    a.polls = kvattn_internal::merge_poll_limit();
    if (lds > 60 * 1024) {
        const int st = hip_status(hipFuncSetAttribute(p.fn, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsMost));
        if (st != KVATTN_OK) return st;
    }
    for (a.row0 = 0; a.row0 < rows; a.row0 += launch_rows) {
        const long long grid = (long long)std::min(launch_rows, rows - a.row0) * p.slices;
        void* params[] = {&a};
        const int st = hip_status(hipLaunchKernel(p.fn, dim3((unsigned)grid), dim3(p.threads), params, lds, (hipStream_t)stream));
        if (st != KVATTN_OK) return st;
    }
    return KVATTN_OK;
}
