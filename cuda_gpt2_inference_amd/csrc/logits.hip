// logits.hip -- rules on logits, and their probabilities, on MI355X (gfx950): penalties for tokens that a sequence
// holds, biases, grammar masks, then the logits or softmax(x / temperature).
//
//   x   = logit; of a token that the sequence holds x / r where positive, else x r      (repetition r)
//   x  -= frequency * count + (count > 0 ? presence : 0)                               (count: times generated)
//   x  += bias;   x = -inf where the grammar forbids the token
//
// A row is one workgroup's: it is read once, stays in registers between the maximum, the sum and the quotient, and is
// written once.  What a sequence holds is a list of ids, so the tokens that any rule names are few against the
// vocabulary: they are set bits of a map in LDS (a bit a token), and a token's place among the set bits, from a
// prefix sum over the map's words, is its entry in a table of counts and biases.  A row's four neighbouring
// tokens look at four bits, and only where one is set at the table.  The row of a token of a tree holds its branch
// too (the bits of its mask), so every row builds its own table.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lanes.hpp"
#include "tree.hpp"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kRun = 4;                        // neighbouring tokens of a thread
constexpr int kStep = kThreads * kRun;         // tokens from one run of a thread to its next
constexpr int kMaxVocab = 1 << 18;
constexpr int kMaxRows = 1 << 21;              // workgroups of a grid: 2^32 threads are too many
constexpr int kMaxSequences = 1 << 20;
constexpr int kLdsMost = 156 * 1024;           // a CU's, less what is static here
constexpr float kLog2e = 1.4426950408889634f;

struct LogitArgs {
    void* out;
    const void* x;
    const int* start;
    kvattn_logit_rules r;
    size_t in_row, out_row;
    int B, rows, V, words, entries;            // words of the map; entries of the table
};

template <bool kF32>
__device__ __forceinline__ float logit(const void* p, size_t i) {
    if constexpr (kF32) return reinterpret_cast<const float*>(p)[i];
    else return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}

template <bool kF32, bool kVec>
__device__ __forceinline__ void load_run(const void* p, size_t row0, int v, int V, float (&x)[kRun]) {
    if (kVec && v + kRun <= V) {
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

template <bool kF32, bool kVec>
__device__ __forceinline__ void store_run(void* p, size_t row0, int v, int V, const float (&x)[kRun]) {
    if (kVec && v + kRun <= V) {
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

// A number that orders as the float does.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// kRuns: runs of a thread that are kept in registers; 0: of a longer row none is, and each pass reads it again.
template <bool kInF32, bool kOutF32, bool kVec, bool kProbs, int kRuns>
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitArgs a) {
    extern __shared__ uint32_t lds[];          // map, its allowed tokens, prefixes (16 bits), counts, biases
    __shared__ uint32_t wave_words[kWaves];
    __shared__ float wave_floats[kWaves];
    __shared__ unsigned long long wave_keys[kWaves];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    constexpr int kHeld = kRuns ? kRuns : 1;
    float x[kHeld][kRun];
    const size_t in0 = (size_t)row * a.in_row, out0 = (size_t)row * a.out_row;
    if constexpr (kRuns > 0) {
#pragma unroll
        for (int j = 0; j < kRuns; ++j) load_run<kInF32, kVec>(a.x, in0, tid * kRun + j * kStep, a.V, x[j]);
    }
    int b = row, t0 = row;
    if (a.start) {
        if (row >= a.start[a.B]) return;       // behind the last token
        b = sequence_of(a.start, a.B, row, lane);
        t0 = min(max(a.start[b], 0), row);
    }

    uint32_t* const map = lds;
    uint32_t* const allowed = map + a.words;
    uint16_t* const before = reinterpret_cast<uint16_t*>(allowed + (a.r.allowed ? a.words : 0));
    uint32_t* const count = reinterpret_cast<uint32_t*>(before) + (a.words + 1) / 2;
    uint32_t* const bias_at = count + a.entries;
    const bool table = a.entries > 0;
    bool grammar = false;
    if (a.r.allowed) {
        const int of = a.r.allowed_of ? a.r.allowed_of[row] : row;
        grammar = of >= 0 && of < a.r.num_allowed;
        if (grammar)
            for (int w = tid; w < a.words; w += kThreads) allowed[w] = a.r.allowed[(size_t)of * a.r.allowed_stride + w];
    }
    if (table) {
        const int held = a.r.history ? min(max(a.r.history_len[b], 0), a.r.max_history) : 0;
        const int prompt = a.r.prompt_len ? a.r.prompt_len[b] : 0;
        const int* const history = a.r.history + (size_t)b * a.r.max_history;
        // This thread's token of the row's branch, and the sequence's biases.
        int branch = -1;
        if (a.r.tokens && tid < 64 * a.r.mask_words && t0 + tid < a.rows) {
            if ((a.r.masks[(size_t)row * a.r.mask_words + (tid >> 6)] >> (tid & 63)) & 1) branch = a.r.tokens[t0 + tid];
        }
        int bias0 = 0, biases = 0;
        if (a.r.bias_start) {
            bias0 = min(max(a.r.bias_start[b], 0), a.r.num_bias);
            biases = min(min(max(a.r.bias_start[b + 1], bias0), a.r.num_bias) - bias0, a.r.max_bias);
        }
        for (int w = tid; w < a.words; w += kThreads) map[w] = 0;
        __syncthreads();
        auto known = [&](int id) { return id >= 0 && id < a.V; };
        auto mark = [&](int id) {
            if (known(id)) atomicOr(map + (id >> 5), 1u << (id & 31));
        };
        for (int i = tid; i < held; i += kThreads) mark(history[i]);
        mark(branch);
        for (int i = tid; i < biases; i += kThreads) mark(a.r.bias_ids[bias0 + i]);
        __syncthreads();
        // Set bits before every word: a thread's words, then the threads'.
        const int per = (a.words + kThreads - 1) / kThreads, w0 = min(tid * per, a.words), w1 = min(w0 + per, a.words);
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
            at += __popc(map[w]);
        }
        for (uint32_t e = tid; e < all; e += kThreads) {
            count[e] = 0;
            if (a.r.bias_start) bias_at[e] = 0;
        }
        __syncthreads();
        auto entry = [&](int id) { return before[id >> 5] + __popc(map[id >> 5] & ((1u << (id & 31)) - 1)); };
        // Times held in the lower half, times of those in the prompt in the upper: at most 2^15 each.
        for (int i = tid; i < held; i += kThreads) {
            const int id = history[i];
            if (known(id)) atomicAdd(count + entry(id), i < prompt ? 0x10001u : 1u);
        }
        if (known(branch)) atomicAdd(count + entry(branch), 1u);
        for (int i = tid; i < biases; i += kThreads) {
            const int id = a.r.bias_ids[bias0 + i];
            if (known(id)) atomicMax(bias_at + entry(id), (uint32_t)(bias0 + i + 1));   // of an id listed twice the last
        }
    }
    const float repetition = a.r.repetition ? a.r.repetition[b] : 1.0f;
    const float frequency = a.r.frequency ? a.r.frequency[b] : 0.0f, presence = a.r.presence ? a.r.presence[b] : 0.0f;
    if (table || a.r.allowed) __syncthreads();

    auto rules = [&](int v, float (&y)[kRun]) {
        if (v >= a.V) return;
        if (table) {
            const uint32_t bits = (map[v >> 5] >> (v & 31)) & 15u;
            if (bits) {
#pragma unroll
                for (int i = 0; i < kRun; ++i) {
#pragma clang fp contract(off)
                    if (!((bits >> i) & 1)) continue;
                    const uint32_t e = before[v >> 5] + __popc(map[v >> 5] & ((1u << ((v + i) & 31)) - 1));
                    const uint32_t c = count[e];
                    const float made = (float)((c & 0xffffu) - (c >> 16));
                    float z = y[i];
                    if (c) z = z > 0.0f ? z / repetition : z * repetition;
                    z = z - (frequency * made + (made > 0.0f ? presence : 0.0f));
                    if (a.r.bias_start) {
                        const uint32_t at = bias_at[e];
                        if (at) z = z + a.r.bias[at - 1];
                    }
                    y[i] = z;
                }
            }
        }
        if (grammar) {
            const uint32_t ok = allowed[v >> 5] >> (v & 31);
#pragma unroll
            for (int i = 0; i < kRun; ++i) y[i] = (ok >> i) & 1 ? y[i] : -INFINITY;
        }
    };
    // Every run of the thread, with the rules applied.
    auto each = [&](auto&& f) {
        if constexpr (kRuns > 0) {
#pragma unroll
            for (int j = 0; j < kRuns; ++j) f(tid * kRun + j * kStep, x[j]);
        } else {
            for (int v = tid * kRun; v < a.V; v += kStep) {
                load_run<kInF32, kVec>(a.x, in0, v, a.V, x[0]);
                rules(v, x[0]);
                f(v, x[0]);
            }
        }
    };
    if constexpr (kRuns > 0) {
#pragma unroll
        for (int j = 0; j < kRuns; ++j) rules(tid * kRun + j * kStep, x[j]);
    }
    if constexpr (!kProbs) {
        each([&](int v, float (&y)[kRun]) { store_run<kOutF32, kVec>(a.out, out0, v, a.V, y); });
        return;
    }
    float top = -INFINITY;
    each([&](int, float (&y)[kRun]) {
#pragma unroll
        for (int i = 0; i < kRun; ++i) top = fmaxf(top, y[i]);
    });
    top = wave_max(top);
    if (lane == 0) wave_floats[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_floats[w]);
    const float temperature = a.r.temperature ? a.r.temperature[b] : 1.0f;
    if (!(temperature > 0.0f) || top == -INFINITY) {
        // The likeliest token alone, the lowest of several; nothing where no token is left.
        unsigned long long best = 0;
        each([&](int v, float (&y)[kRun]) {
#pragma unroll
            for (int i = 0; i < kRun; ++i) {
                const unsigned long long key = (unsigned long long)ordered(y[i]) << 32 | (0xffffffffu - (uint32_t)(v + i));
                if (y[i] == top && v + i < a.V && key > best) best = key;
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
        const int token = top == -INFINITY ? -1 : (int)(0xffffffffu - (uint32_t)best);
        each([&](int v, float (&y)[kRun]) {
#pragma unroll
            for (int i = 0; i < kRun; ++i) y[i] = v + i == token ? 1.0f : 0.0f;
            store_run<kOutF32, kVec>(a.out, out0, v, a.V, y);
        });
        return;
    }
    const float scale = kLog2e / temperature;
    auto weigh = [&](float (&y)[kRun]) {
#pragma unroll
        for (int i = 0; i < kRun; ++i) y[i] = exp2_fast((y[i] - top) * scale);
    };
    float sum = 0.0f;
    each([&](int, float (&y)[kRun]) {
        weigh(y);
        sum += (y[0] + y[1]) + (y[2] + y[3]);
    });
    sum = wave_sum(sum);
    __syncthreads();                           // (the maxima have been read)
    if (lane == 0) wave_floats[wave] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += wave_floats[w];
    const float one = 1.0f / sum;
    each([&](int v, float (&y)[kRun]) {
        if constexpr (kRuns == 0) weigh(y);
        // (A forbidden token has none, also where the others' is NaN.)
#pragma unroll
        for (int i = 0; i < kRun; ++i) y[i] = y[i] == 0.0f ? 0.0f : y[i] * one;
        store_run<kOutF32, kVec>(a.out, out0, v, a.V, y);
    });
}

template <bool kInF32, bool kOutF32, bool kVec, bool kProbs>
const void* kernel_for(int V) {
    if (V <= 4 * kStep) return (const void*)&logits_kernel<kInF32, kOutF32, kVec, kProbs, 4>;
    if (V <= 13 * kStep) return (const void*)&logits_kernel<kInF32, kOutF32, kVec, kProbs, 13>;
    return (const void*)&logits_kernel<kInF32, kOutF32, kVec, kProbs, 0>;
}
template <bool kInF32, bool kOutF32>
const void* kernel_for(int V, bool vec, bool probs) {
    if (vec) return probs ? kernel_for<kInF32, kOutF32, true, true>(V) : kernel_for<kInF32, kOutF32, true, false>(V);
    return probs ? kernel_for<kInF32, kOutF32, false, true>(V) : kernel_for<kInF32, kOutF32, false, false>(V);
}

int hip_status(hipError_t e) {
    if (e == hipSuccess) return KVATTN_OK;
    kvattn_internal::set_last_hip_error((int)e);
    return KVATTN_ERR_HIP;
}

}  // namespace

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
    if (((uintptr_t)r.masks & 7u) || ((uintptr_t)logits % in) || ((uintptr_t)out % res)) return KVATTN_ERR_MISALIGNED;
    if (r.bias_start && (r.num_bias == 0 || r.max_bias == 0)) r.bias_start = nullptr;
    a.out = out;
    a.x = logits;
    a.start = token_start;
    a.in_row = (size_t)row_stride;
    a.out_row = (size_t)out_stride;
    a.B = B;
    a.rows = rows;
    a.V = V;
    a.words = (V + 31) / 32;
    // Every entry is another token: a row has no more of them than of these.
    a.entries = std::min(V, (r.history ? r.max_history : 0) + (branches ? 64 * r.mask_words : 0) + (r.bias_start ? r.max_bias : 0));
    const size_t lds = (size_t)a.words * (r.allowed ? 8 : 4) + (size_t)(a.words + 1) / 2 * 4 + (size_t)a.entries * (r.bias_start ? 8 : 4);
    if (lds > kLdsMost) return KVATTN_ERR_LDS;
    const bool vec = row_stride % kRun == 0 && out_stride % kRun == 0 && ((uintptr_t)logits % (kRun * in)) == 0 &&
                     ((uintptr_t)out % (kRun * res)) == 0;
    const void* fn = dtype == KVATTN_KV_F32 ? (out_dtype == KVATTN_KV_F32 ? kernel_for<true, true>(V, vec, probs != 0) : kernel_for<true, false>(V, vec, probs != 0))
                                            : (out_dtype == KVATTN_KV_F32 ? kernel_for<false, true>(V, vec, probs != 0) : kernel_for<false, false>(V, vec, probs != 0));
    if (lds > 64 * 1024 - 512) {
        const int st = hip_status(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsMost));
        if (st != KVATTN_OK) return st;
    }
    void* params[] = {&a};
    return hip_status(hipLaunchKernel(fn, dim3((unsigned)rows), dim3(kThreads), params, lds, (hipStream_t)stream));
}
