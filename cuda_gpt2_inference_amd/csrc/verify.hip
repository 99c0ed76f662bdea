// verify.hip -- verification of drafted tokens on MI355X (gfx950): a sequence's drafts are accepted
// one after another while r q(x) < p(x), and the token behind the last accepted one is drawn from
// max(0, p - q) where a draft was refused, from p where none was, by the inverse of the running sum.
//
// Only one row of p and one of q a sequence is read whole (2 x 200 KB at GPT-2's vocabulary): which
// one follows from a few single values, which every wave looks up for itself.  The row is cut into
// tiles of 1024 tokens; a wave sums one at a time, then one wave finds the tile that the random number
// falls into and the token in it.  Sums are double: a running float sum over 50,000 tokens would move
// the border between two tokens by more than most tokens' whole probability.
//
// Bound by a chain of dependent memory round trips (offsets, drafts, their probabilities, the row, the
// sums, the tile).  Workgroups of a sequence run on one XCD, so that the values that each of them looks
// up, and the tile that is read again, come from its L2.  One workgroup of 16 waves a sequence, whose
// sums stay in LDS, saves the join's round trips but draws the row through one CU: 19 us against 8 for
// one sequence, 32 against 13 for 64 (before the steps below).  A wave's arithmetic counts next to the round trips:
// a weight of five instructions in place of eight, and the drawn token's tile divided among four
// waves, took one sequence from 7.2 to 5.8 us, 64 from 11.3 to 10.2.  Workgroups of 4 / 8 / 16 waves:
// one sequence 5.6 / 5.8 / 6.3 us, 64 of them 10.5 / 10.2 / 9.5, 300 19.6 / 19.2 / 20.8.  One / two workgroups
// a CU: 64 10.6 / 10.5, 300 21.6 / 19.4.
#include <hip/hip_runtime.h>

#include "kvattn.h"
#include "lanes.hpp"

namespace kvattn_internal {
void set_last_hip_error(int e);   // kvattn.hip: read back by kvattn_last_hip_error
}

namespace {

constexpr int kBlock = 512;
constexpr int kWaves = kBlock / kWave;
constexpr int kTile = 16 * kWave;         // tokens of a wave's tile: 16 a lane
constexpr int kRuns = 4;                  // runs of a tile: neighbouring tokens of all lanes
static_assert(kWaves >= kRuns && kTile == kRuns * 4 * kWave, "a wave for every run");
constexpr int kMaxVocab = 1 << 24;
constexpr int kMaxSequences = 1 << 16;
constexpr int kMostTokens = 1 << 30;      // a wave's next 64 drafts beyond are still an int
constexpr int kFillBlocks = 512;          // workgroups that keep the memory busy, two a CU

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

// Four neighbouring probabilities from token v on.
template <bool kF32>
__device__ __forceinline__ void probs4(const void* p, size_t row0, int v, float* x) {
    if constexpr (kF32) {
        const float4 w = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + row0 + v);
        x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + row0 + v);
        x[0] = bf16_lo(w.x); x[1] = bf16_hi(w.x); x[2] = bf16_lo(w.y); x[3] = bf16_hi(w.y);
    }
}

// A lane's probabilities of a tile: four neighbours from token_at on in each of its four runs, where they
// lie next to the neighbouring lanes'.  Zero past the vocabulary.  The branch is the wave's, so that all
// of the loads are on their way at once.
__device__ __forceinline__ int token_at(int tile, int run, int lane) { return tile * kTile + (run * kWave + lane) * 4; }
template <bool kF32, bool kVec>
__device__ __forceinline__ void run_probs(const void* p, size_t row0, int tile, int run, int V, int lane, float* x) {
    const int v0 = token_at(tile, run, lane);
    if (kVec && tile * kTile + kTile <= V) {
        probs4<kF32>(p, row0, v0, x);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float w = prob<kF32>(p, row0 + min(v0 + i, V - 1));
        x[i] = v0 + i < V ? w : 0.0f;
    }
}
template <bool kF32, bool kVec>
__device__ __forceinline__ void tile_probs(const void* p, size_t row0, int tile, int V, int lane, float (&x)[16]) {
    if (kVec && tile * kTile + kTile <= V) {
#pragma unroll
        for (int j = 0; j < 4; ++j) probs4<kF32>(p, row0, token_at(tile, j, lane), x + 4 * j);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) run_probs<kF32, false>(p, row0, tile, j, V, lane, x + 4 * j);
}

// What a token weighs: a positive number, or nothing; NaN, which what is not finite becomes (x + 0 x), nothing.
__device__ __forceinline__ double finite(float x) { return (double)fmaf(x, 0.0f, x); }
__device__ __forceinline__ double mass(double w) { return fmax(w, 0.0); }

// Sums across lanes through DPP, as the float ones: a shuffle's trip through LDS in each of the six
// steps of four sums added up to a microsecond.
template <int kCtrl, int kRows = 0xF>
__device__ __forceinline__ double dpp64(double x) {      // lanes without a source, or outside kRows, get zero
    const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, kCtrl, kRows, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), kCtrl, kRows, 0xF, true);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
template <bool k32>
__device__ __forceinline__ double add_across(double x) { // x + x of lane ^ 16 or ^ 32
    const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
    const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
    const auto l = k32 ? __builtin_amdgcn_permlane32_swap(lo, lo, false, false) : __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    const auto h = k32 ? __builtin_amdgcn_permlane32_swap(hi, hi, false, false) : __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    return __builtin_bit_cast(double, (unsigned long long)h[0] << 32 | l[0]) +
           __builtin_bit_cast(double, (unsigned long long)h[1] << 32 | l[1]);
}
__device__ __forceinline__ double wave_sum64(double x) {
    x += dpp64<kDppQuadXor1>(x);
    x += dpp64<kDppQuadXor2>(x);
    x += dpp64<kDppHalfMirror>(x);
    x += dpp64<kDppRowMirror>(x);
    return add_across<true>(add_across<false>(x));
}

// Inclusive prefix over the wave's lanes: rows of 16 by shifts, then the last lane of the row before into
// rows 1 and 3, and lane 31 into the upper two.
__device__ __forceinline__ double wave_prefix64(double x) {
    x += dpp64<0x111>(x);                  // row_shr:1, 2, 4, 8
    x += dpp64<0x112>(x);
    x += dpp64<0x114>(x);
    x += dpp64<0x118>(x);
    x += dpp64<0x142, 0xA>(x);             // row_bcast:15
    x += dpp64<0x143, 0xC>(x);             // row_bcast:31
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
    __shared__ double run_sums[kRuns];
    const int slot = xcd_slot(blockIdx.x, a.blocks), b = slot / a.blocks, blk = slot - b * a.blocks;
    if (b >= a.B) return;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int t0 = min(max(a.start[b], 0), a.num_tokens);
    const int n = min(max(a.start[b + 1], t0), a.num_tokens) - t0;
    if (n == 0) {
        if (blk == 0 && threadIdx.x == 0) a.count[b] = 0;
        return;
    }
    const float u_last = a.u[t0 + n - 1];  // a number that no draft is held against
    // The first row whose draft is not accepted (the last row has none): 64 rows at a time, a lane
    // each.  The comparison is exact: products of two floats fit a double.
    int row = n - 1, draft = -1;
    for (int i0 = 0; i0 < n - 1; i0 += kWave) {
        const int i = i0 + lane;
        bool no = false;
        int x = -1;
        if (i < n - 1) {
            x = a.drafts[t0 + i];
            const size_t at = (size_t)(t0 + i) * a.row + x;
            no = !(x >= 0 && x < a.V);
            if (!no) {
                const double q = a.q ? (double)prob<kF32>(a.q, at) : 1.0;
                no = !((double)a.u[t0 + i] * q < (double)prob<kF32>(a.p, at));
            }
        }
        const unsigned long long refused = __ballot(no);
        if (refused) {
            const int at = __ffsll((long long)refused) - 1;
            row = i0 + at;
            draft = __builtin_amdgcn_readlane(x, at);
            break;
        }
    }
    const bool refused = row < n - 1;
    const bool less_q = refused && a.q;
    const size_t row0 = (size_t)(t0 + row) * a.row;

    for (int tile = blk * kWaves + wave; tile < a.tiles; tile += a.blocks * kWaves) {
        float p[16], q[16];
        tile_probs<kF32, kVec>(a.p, row0, tile, a.V, lane, p);
        if (less_q) tile_probs<kF32, kVec>(a.q, row0, tile, a.V, lane, q);
        double rest = 0.0, all = 0.0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const double w = finite(p[e]);
            all += mass(w);
            if (less_q) rest += mass(w - finite(q[e]));
        }
        // A draft without probabilities had it all, and leaves its own token nothing.
        if (!less_q) {
            rest = all;
            if (draft >= 0 && draft / kTile == tile) {
                rest = 0.0;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    rest += token_at(tile, e / 4, lane) + e % 4 == draft ? 0.0 : mass(finite(p[e]));
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
    wait_vm_stores();
    __syncthreads();
    if (threadIdx.x == 0 && a.blocks == 1) is_last = 1;
    if (threadIdx.x == 0 && a.blocks > 1) {
        const unsigned before = __hip_atomic_fetch_add(a.counters + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        is_last = before == (unsigned)(a.blocks - 1);
        if (is_last) __hip_atomic_store(a.counters + b, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!is_last) return;
    if (wave >= kRuns) return;

    // Totals, and which weights count: where a refused draft leaves nothing (p = q), p's own.
    const double* const s = a.sums + (size_t)b * a.tiles * 2;
    auto sums_at = [&](int t, double& r, double& l) {
        const int at = min(t, a.tiles - 1);
        r = get64(s + 2 * at);
        l = get64(s + 2 * at + 1);
        if (t >= a.tiles) r = l = 0.0;
    };
    double rest0, all0, rest, all;         // of tile lane, kept; of every 64th from there
    sums_at(lane, rest0, all0);
    rest = rest0;
    all = all0;
    for (int t = lane + kWave; t < a.tiles; t += kWave) {
        double r, l;
        sums_at(t, r, l);
        rest += r;
        all += l;
    }
    rest = wave_sum64(rest);
    all = wave_sum64(all);
    const bool use_rest = rest > 0.0;
    const double total = use_rest ? rest : all;
    const double aim = (double)u_last * total;
    int drawn = -1;
    // The sums are left at zero, as the counter is, once all four waves have read them: where they lie,
    // a call of another B or V has its counters.
    auto leave_zero = [&] {
        __syncthreads();
        double* const z = a.sums + (size_t)b * a.tiles * 2;
        for (int t = threadIdx.x; t < 2 * a.tiles; t += kRuns * kWave) put64(z + t, 0.0);
    };
    if (total > 0.0) {
        // The first tile whose running sum passes the aim (rounding may leave none: the last that weighs
        // anything), then the first run of it, then the first token likewise.
        int tile = -1;
        double base = 0.0, before = 0.0;
        for (int t1 = 0; t1 < a.tiles; t1 += kWave) {
            double r = rest0, l = all0;
            if (t1 > 0) sums_at(t1 + lane, r, l);
            const double w = use_rest ? r : l;
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
        // Every wave takes one of the tile's runs; the one that the aim falls into goes on.
        float p[4], q[4];
        run_probs<kF32, kVec>(a.p, row0, tile, wave, a.V, lane, p);
        if (use_rest && less_q) run_probs<kF32, kVec>(a.q, row0, tile, wave, a.V, lane, q);
        const int v0 = token_at(tile, wave, lane);
        double w[4], mine = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = finite(p[i]);
            if (use_rest && less_q) w[i] -= finite(q[i]);
            w[i] = use_rest && !less_q && v0 + i == draft ? 0.0 : mass(w[i]);
            mine += w[i];
        }
        const double sum = wave_prefix64(mine);
        if (lane == kWave - 1) run_sums[wave] = sum;
        leave_zero();
        int run = -1;
        double run0 = 0.0;
        bool passed = false;
#pragma unroll
        for (int j = 0; j < kRuns; ++j) {
            const double r = run_sums[j];
            if (r > 0.0 && !passed) {
                run = j;
                run0 = base;
                passed = base + r > aim;
            }
            base += r;
        }
        if (wave != run) return;
        double upto = run0 + (sum - mine);
        int hit = -1, last = -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            upto += w[i];
            if (w[i] > 0.0) {
                last = v0 + i;
                if (hit < 0 && upto > aim) hit = last;
            }
        }
        const unsigned long long pass = __ballot(hit >= 0), some = __ballot(last >= 0);
        if (pass) drawn = __shfl(hit, __ffsll((long long)pass) - 1);
        else if (some) drawn = __shfl(last, 63 - __clzll((long long)some));
    } else {
        leave_zero();
        if (wave != 0) return;
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
    if (B < 1 || B > kMaxSequences || V < 1 || V > kMaxVocab || num_tokens < 0 || num_tokens > kMostTokens || row_stride < V)
        return KVATTN_ERR_SHAPE;
    if (!counts || !token_start) return KVATTN_ERR_NULL_POINTER;
    // (Nothing of an array without elements is looked at, and its address may be none.)
    if (num_tokens > 0 && (!tokens || !target_probs || !draft_tokens || !uniform)) return KVATTN_ERR_NULL_POINTER;
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
    const long long grid = 8ll * ((B + 7) / 8) * a.blocks;      // whole rounds of the eight XCDs
    void* params[] = {&a};
    const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)grid), dim3(kBlock), params, 0,
                                         (hipStream_t)stream);
    if (e != hipSuccess) {
        kvattn_internal::set_last_hip_error((int)e);
        return KVATTN_ERR_HIP;
    }
    return KVATTN_OK;
}

}  // extern "C"
