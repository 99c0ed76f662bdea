// verify.hip -- verification of drafted tokens on MI355X (gfx950): a sequence's drafts are accepted
// one after another while r q(x) < p(x), and the token behind the last accepted one is drawn from
// max(0, p - q) where a draft was refused, from p where none was, by the inverse of the running sum.
//
// Only one row of p and one of q a sequence is read whole (2 x 200 KB at GPT-2's vocabulary): which
// one follows from a few single values, which every workgroup of a sequence looks up for itself.
// The row is cut into tiles of 1024 tokens, one a wave; their sums go to the workspace, and the
// workgroup that finishes last finds the tile that the random number falls into and then the token
// in it.  One launch, bound by memory for batches and by four dependent round trips for one
// sequence.  Sums are double: a running float sum over 50,000 tokens would move the border between
// two tokens by more than most tokens' whole probability.
#include <hip/hip_runtime.h>

#include "kvattn.h"
#include "lanes.hpp"

namespace kvattn_internal {
void set_last_hip_error(int e);   // kvattn.hip: read back by kvattn_last_hip_error
}

namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr int kTile = 1024;               // tokens of a wave's tile: 16 a lane
constexpr int kMaxVocab = 1 << 24;
constexpr int kMaxSequences = 1 << 16;
constexpr int kFillBlocks = 1024;         // workgroups that keep the memory busy

struct VerifyArgs {
    int* tokens;
    int* count;
    const void* p;
    const void* q;
    const int* drafts;
    const float* u;
    const int* start;
    double* sums;                         // [B][tiles][2]: of max(0, p - q), of p
    unsigned* counters;
    size_t row;                           // elements from one row to the next
    int B, num_tokens, V, tiles, blocks;  // blocks: workgroups of a sequence
};

template <bool kF32>
__device__ __forceinline__ float prob(const void* p, size_t i) {
    if constexpr (kF32) return reinterpret_cast<const float*>(p)[i];
    else return bf16_to_f32(reinterpret_cast<const uint16_t*>(p)[i]);
}

// Four neighbouring probabilities from token v on; zero past the vocabulary.
template <bool kF32, bool kVec>
__device__ __forceinline__ void probs4(const void* p, size_t row0, int v, int V, float (&x)[4]) {
    if (kVec && v + 3 < V) {
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
    for (int i = 0; i < 4; ++i) x[i] = v + i < V ? prob<kF32>(p, row0 + v + i) : 0.0f;
}

// What a token weighs: a finite positive number, or nothing.
__device__ __forceinline__ double mass(double w) { return w > 0.0 && w < INFINITY ? w : 0.0; }

__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) x += __shfl_xor(x, d);
    return x;
}

// Inclusive prefix over the wave's lanes.
__device__ __forceinline__ double wave_prefix64(double x) {
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const double o = __shfl_up(x, d);
        x += lane >= d ? o : 0.0;
    }
    return x;
}

__device__ __forceinline__ void put64(double* p, double v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get64(const double* p) {
    return __hip_atomic_load(const_cast<double*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <bool kF32, bool kVec>
__global__ __launch_bounds__(kBlock) void verify_kernel(VerifyArgs a) {
    __shared__ int is_last;
    const int b = blockIdx.x / a.blocks, blk = blockIdx.x - b * a.blocks;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int t0 = min(max(a.start[b], 0), a.num_tokens);
    const int n = min(max(a.start[b + 1], t0), a.num_tokens) - t0;
    if (n == 0) {
        if (blk == 0 && threadIdx.x == 0) a.count[b] = 0;
        return;
    }
    // The first row whose draft is not accepted (the last row has none): 64 rows at a time, a lane
    // each.  The comparison is exact: products of two floats fit a double.
    int row = n - 1;
    for (int i0 = 0; i0 < n - 1; i0 += kWave) {
        const int i = i0 + lane;
        bool no = false;
        if (i < n - 1) {
            const int x = a.drafts[t0 + i];
            const size_t at = (size_t)(t0 + i) * a.row + x;
            no = !(x >= 0 && x < a.V);
            if (!no) {
                const double q = a.q ? (double)prob<kF32>(a.q, at) : 1.0;
                no = !((double)a.u[t0 + i] * q < (double)prob<kF32>(a.p, at));
            }
        }
        const unsigned long long refused = __ballot(no);
        if (refused) {
            row = i0 + __ffsll((long long)refused) - 1;
            break;
        }
    }
    const bool refused = row < n - 1;
    const int draft = refused ? a.drafts[t0 + row] : -1;
    const bool less_q = refused && a.q;
    const size_t row0 = (size_t)(t0 + row) * a.row;

    // Four tokens' weights: with the draft's distribution taken off, or without.
    auto weights = [&](int v, bool rest, double (&w)[4]) {
        float p[4], q[4];
        probs4<kF32, kVec>(a.p, row0, v, a.V, p);
        if (rest && less_q) probs4<kF32, kVec>(a.q, row0, v, a.V, q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = (double)p[i];
            if (rest && less_q) w[i] -= (double)q[i];
            else if (rest && v + i == draft) w[i] = 0.0;      // a draft without probabilities had it all
            w[i] = mass(w[i]);
        }
    };

    for (int tile = blk * kWaves + wave; tile < a.tiles; tile += a.blocks * kWaves) {
        double rest = 0.0, all = 0.0;
#pragma unroll
        for (int j = 0; j < kTile / (4 * kWave); ++j) {
            const int v = tile * kTile + (j * kWave + lane) * 4;
            float p[4], q[4];
            probs4<kF32, kVec>(a.p, row0, v, a.V, p);
            if (less_q) probs4<kF32, kVec>(a.q, row0, v, a.V, q);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                all += mass((double)p[i]);
                if (less_q) rest += mass((double)p[i] - (double)q[i]);
                else if (v + i != draft) rest += mass((double)p[i]);
            }
        }
        rest = wave_sum64(rest);
        all = wave_sum64(all);
        if (lane == 0) {
            double* const s = a.sums + ((size_t)b * a.tiles + tile) * 2;
            put64(s, rest);
            put64(s + 1, all);
        }
    }
    if (a.blocks > 1) {
        wait_vm_stores();
        __syncthreads();
        if (threadIdx.x == 0) {
            const unsigned before = __hip_atomic_fetch_add(a.counters + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            is_last = before == (unsigned)(a.blocks - 1);
            if (is_last) __hip_atomic_store(a.counters + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!is_last) return;
    } else {
        wait_vm_stores();
        __syncthreads();
    }
    if (wave != 0) return;

    // Totals, and which weights count: where a refused draft leaves nothing (p = q), p's own.
    const double* const s = a.sums + (size_t)b * a.tiles * 2;
    double rest = 0.0, all = 0.0;
    for (int t = lane; t < a.tiles; t += kWave) {
        rest += get64(s + 2 * t);
        all += get64(s + 2 * t + 1);
    }
    rest = wave_sum64(rest);
    all = wave_sum64(all);
    const bool use_rest = rest > 0.0;
    const double total = use_rest ? rest : all;
    const double aim = (double)a.u[t0 + n - 1] * total;   // a number that no draft was held against
    int drawn = -1;
    if (total > 0.0) {
        // The first tile whose running sum passes the aim (rounding may leave none: the last that weighs
        // anything), then the first token in it likewise.
        int tile = -1;
        double base = 0.0, before = 0.0;
        for (int t1 = 0; t1 < a.tiles; t1 += kWave) {
            const int t = t1 + lane;
            const double w = t < a.tiles ? get64(s + 2 * t + (use_rest ? 0 : 1)) : 0.0;
            const double upto = before + wave_prefix64(w);
            const unsigned long long pass = __ballot(w > 0.0 && upto > aim), some = __ballot(w > 0.0);
            if (some) {
                const int at = pass ? __ffsll((long long)pass) - 1 : 63 - __clzll((long long)some);
                tile = t1 + at;
                base = __shfl(upto - w, at);
            }
            if (pass) break;
            before = __shfl(upto, kWave - 1);
        }
        for (int j = 0; j < kTile / (4 * kWave); ++j) {
            const int v = tile * kTile + (j * kWave + lane) * 4;
            double w[4];
            weights(v, use_rest, w);
            const double mine = (w[0] + w[1]) + (w[2] + w[3]);
            const double upto = base + wave_prefix64(mine);
            double run = upto - mine;
            int hit = -1, last = -1;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                run += w[i];
                if (w[i] > 0.0) {
                    last = v + i;
                    if (hit < 0 && run > aim) hit = v + i;
                }
            }
            const unsigned long long pass = __ballot(hit >= 0), some = __ballot(last >= 0);
            if (pass) {
                drawn = __shfl(hit, __ffsll((long long)pass) - 1);
                break;
            }
            if (some) drawn = __shfl(last, 63 - __clzll((long long)some));
            base = __shfl(upto, kWave - 1);
        }
    }
    for (int i = lane; i < n; i += kWave) a.tokens[t0 + i] = i < row ? a.drafts[t0 + i] : (i == row ? drawn : -1);
    if (lane == 0) a.count[b] = row + (drawn >= 0 ? 1 : 0);
}

int tiles_of(int V) { return (V + kTile - 1) / kTile; }
size_t up256(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace

extern "C" {

size_t kvattn_verify_workspace_bytes(int B, int V) {
    if (B < 1 || B > kMaxSequences || V < 1 || V > kMaxVocab) return 0;
    return up256((size_t)B * sizeof(unsigned)) + up256((size_t)B * tiles_of(V) * 2 * sizeof(double));
}

int kvattn_verify_drafts(int* tokens, int* counts, const void* target_probs, const void* draft_probs,
                         const int* draft_tokens, const float* uniform, const int* token_start, int B, int num_tokens,
                         int V, long long row_stride, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (dtype != KVATTN_KV_F32 && dtype != KVATTN_KV_BF16) return KVATTN_ERR_DTYPE;
    if (B < 1 || B > kMaxSequences || V < 1 || V > kMaxVocab || num_tokens < 0 || row_stride < V) return KVATTN_ERR_SHAPE;
    if (!tokens || !counts || !target_probs || !draft_tokens || !uniform || !token_start) return KVATTN_ERR_NULL_POINTER;
    const size_t size = dtype == KVATTN_KV_F32 ? 4 : 2;
    if (((uintptr_t)target_probs % size) || ((uintptr_t)draft_probs % size) || ((uintptr_t)tokens & 3u) ||
        ((uintptr_t)counts & 3u) || ((uintptr_t)draft_tokens & 3u) || ((uintptr_t)uniform & 3u) ||
        ((uintptr_t)token_start & 3u) || ((uintptr_t)workspace & 255u))
        return KVATTN_ERR_MISALIGNED;
    if (!workspace || workspace_bytes < kvattn_verify_workspace_bytes(B, V)) return KVATTN_ERR_WORKSPACE;
    VerifyArgs a{};
    a.tokens = tokens;
    a.count = counts;
    a.p = target_probs;
    a.q = draft_probs;
    a.drafts = draft_tokens;
    a.u = uniform;
    a.start = token_start;
    a.counters = (unsigned*)workspace;
    a.sums = (double*)((uint8_t*)workspace + up256((size_t)B * sizeof(unsigned)));
    a.row = (size_t)row_stride;
    a.B = B;
    a.num_tokens = num_tokens;
    a.V = V;
    a.tiles = tiles_of(V);
    const int most = (a.tiles + kWaves - 1) / kWaves;      // one tile a wave
    const int few = (kFillBlocks + B - 1) / B;
    a.blocks = most < few ? most : few;
    // Four probabilities in one load where every row starts on such a boundary.
    const bool vec = row_stride % 4 == 0 && ((uintptr_t)target_probs % (4 * size)) == 0 &&
                     ((uintptr_t)draft_probs % (4 * size)) == 0;
    const void* fn = dtype == KVATTN_KV_F32
                         ? (vec ? (const void*)&verify_kernel<true, true> : (const void*)&verify_kernel<true, false>)
                         : (vec ? (const void*)&verify_kernel<false, true> : (const void*)&verify_kernel<false, false>);
    void* params[] = {&a};
    const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)((long long)a.blocks * B)), dim3(kBlock), params, 0,
                                         (hipStream_t)stream);
    if (e != hipSuccess) {
        kvattn_internal::set_last_hip_error((int)e);
        return KVATTN_ERR_HIP;
    }
    return KVATTN_OK;
}

}  // extern "C"
