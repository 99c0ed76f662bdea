// pages.hip -- the bookkeeping of a paged KV cache on the GPU, and its rows by slot map (gfx950):
// block tables, token offsets, slot map and positions from what every request holds, keeps and
// adds; K and V rows into the pool and out of it for every cache type; the append of one token a
// sequence into a 4-bit cache.
#include "kv4.hpp"

#include <limits.h>

#include "lanes.hpp"
#include "layout.hpp"

namespace {

using kvattn_internal::is_4bit;

constexpr int kHd = 64;
constexpr int kBlock = 256;
constexpr int kMaxT = 1 << 23;

int log2_or(int x) { return x > 0 && (x & (x - 1)) == 0 ? __builtin_ctz((unsigned)x) : -1; }

int hip_status(hipError_t e) {
    if (e == hipSuccess) return KVATTN_OK;
    kvattn_internal::set_last_hip_error((int)e);
    return KVATTN_ERR_HIP;
}

// ------------------------------------------------------------------------------------
// Pages of requests.
//
// The pool is a ring of free page ids: taken at its head, given back at its tail, so a call's
// reads (entries head ..) and writes (entries head + count ..) never meet.  Every workgroup reads
// all requests and scans them (tokens, pages taken, pages given back: prefix sums in request
// order), then does its share of the tokens and pages, which need nothing of one another.  What the
// outputs may share with the inputs (held, kept, the pool's head and count) is written by the
// workgroup that was the last to have read it all, so one launch does, in place too.  24 requests (3.7 us,
// 2.2 an empty graph node) are bound by three memory round trips; 1000 with 250,000 tokens (7.7 us) by the
// scan, 2.1 us, every token's lookup, 1.8, and the last workgroup's turn, 0.9.
// ------------------------------------------------------------------------------------
constexpr int kPoolHead = 0, kPoolCount = 1, kPoolTicket = 2, kPoolRing = 4;
constexpr int kMaxRequests = 4096;
constexpr int kRequestInts = 6;            // LDS words of a request
constexpr int kReserveThreads = 1024;      // of a workgroup; kSmallThreads where one such is enough
constexpr int kSmallThreads = 256;
constexpr int kReserveTokens = 4096;       // token rows a workgroup is launched for, up to
constexpr int kReserveMostBlocks = 256;    // so many workgroups
constexpr int kMostTokens = 1 << 30;       // a step of every workgroup's threads beyond is still an int
constexpr int kRefused = 1 << 30;          // beside the positions a request keeps

struct ReserveArgs {
    int* table;
    int* pool;
    const int* held;
    const int* kept;
    const int* fresh;
    int* held_out;
    int* lens;
    int* token_start;
    long long* slot_map;
    int* positions;
    int* pool_next;
    int max_pages, R, num_pages, B, max_tokens;
    int shift;                 // log2 of R, or -1
    int grid;                  // workgroups
};

__device__ __forceinline__ int add_sat(int a, int b) {   // a, b >= 0
    const unsigned s = (unsigned)a + (unsigned)b;
    return s > (unsigned)INT_MAX ? INT_MAX : (int)s;
}

// Inclusive prefix over the wave's lanes (saturating; values >= 0): rows of 16 by shifts, then the last
// lane of the row before into rows 1 and 3, and lane 31 into the upper two.
__device__ __forceinline__ int wave_prefix(int x) {
    x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true));   // row_shr:1, 2, 4, 8
    x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true));
    x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true));
    x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true));
    x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, true));   // row_bcast:15
    x = add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, true));   // row_bcast:31
    return x;
}

// A barrier for what was written to LDS: global reads and writes stay on their way (__syncthreads waits for them).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The largest over the wave's lanes (values >= 0), in every lane.
__device__ __forceinline__ int wave_top(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, true));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, true));
    return __builtin_amdgcn_readlane(x, kWave - 1);
}

// Exclusive prefixes of kN values over the workgroup's threads (kAlone: the wave's), and their totals.  Subtraction undoes a
// sum only where nothing was cut off, so the values themselves are shifted by a lane.
template <int kThreads, bool kAlone, int kN>
__device__ __forceinline__ void prefix_of(const int (&v)[kN], int (&wave_sums)[kN][kThreads / kWave], int (&prefix)[kN],
                                             int (&total)[kN]) {
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    int in[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        in[n] = wave_prefix(v[n]);
        if (!kAlone && lane == kWave - 1) wave_sums[n][wave] = in[n];
    }
    if (!kAlone) lds_barrier();
    // The waves' sums: a prefix over the first lanes of every wave.
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        const int upto = kAlone ? in[n] : wave_prefix(lane < kThreads / kWave ? wave_sums[n][lane] : 0);
        const int before = !kAlone && wave > 0 ? __builtin_amdgcn_readlane(upto, wave - 1) : 0;
        const int up = __shfl_up(in[n], 1);
        prefix[n] = add_sat(before, lane > 0 ? up : 0);
        total[n] = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
}

// The last i of lo .. hi with start[i] <= x (start[lo] <= x): the owner of item x.
__device__ __forceinline__ int owner(const int* start, int lo, int hi, int x) {
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// The same for an x that the wave's lanes share, over all of n entries: 64 of them looked at at once.
__device__ __forceinline__ int owner_of(const int* start, int n, int x) {
    const int lane = threadIdx.x & (kWave - 1);
    int lo = 0;
    for (int step = n > kWave ? kWave : 1;; step = 1) {
        const int i = lo + lane * step;
        const unsigned long long at = __ballot(i < n && start[min(i, n - 1)] <= x);
        lo += (63 - __clzll((long long)(at | 1))) * step;
        if (step == 1) return lo;
    }
}

// kEach: kMany; kOne: no more requests than threads, so that a thread's own one stays in its registers;
// kWaves: no more than lanes, and every wave does all of them for itself, with a copy in LDS of its own,
// so that nobody waits for anybody (24 requests 4.1 us, 3.7 so).
enum Each { kMany, kOne, kWaves };
template <int kThreads, int kEach>
__global__ __launch_bounds__(kThreads) void reserve_kernel(ReserveArgs a) {
    extern __shared__ int lds[];
    __shared__ int asked_sums[2][kThreads / kWave], given_sums[1][kThreads / kWave];
    __shared__ int took_sums[kThreads / kWave], shared_turn;
    constexpr int kOwn = kEach == kMany ? kMaxRequests / kThreads : 1;   // requests a thread reads
    const int tid = threadIdx.x, self = kEach == kWaves ? tid & (kWave - 1) : tid;
    int* const tok = lds + (kEach == kWaves ? tid / kWave * kRequestInts * a.B : 0);   // first token
    int* const take = tok + a.B;          // first of the pages it takes
    int* const give = take + a.B;         // first of the pages it gives back
    int* const have = give + a.B;         // pages it holds
    int* const want = have + a.B;         // pages it will hold (refused: those it holds)
    int* const kept = want + a.B;         // positions it keeps, and kRefused
    const int P = a.num_pages;
    const int head = (int)((unsigned)a.pool[kPoolHead] % (unsigned)P);
    const int count = min(max(a.pool[kPoolCount], 0), P);
    const long long most = (long long)a.max_pages * a.R;
    auto pages_of = [&](int positions) {
        return a.shift >= 0 ? (positions + a.R - 1) >> a.shift : (positions + a.R - 1) / a.R;
    };
    // A request's tokens and pages; one whose lengths make no sense asks for nothing.
    struct Request {
        int tok, have, want, kept;
    };
    int hd_own[kOwn], kp_own[kOwn];
    Request own = {0, 0, 0, kRefused};
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int i = self + j * kThreads;
        if (i >= a.B) break;
        const int hd = a.held[i], kp = a.kept[i], fr = a.fresh[i];
        hd_own[j] = hd;
        kp_own[j] = kp;
        const bool ok = kp >= 0 && kp <= hd && hd <= most && fr >= 0 && (long long)kp + fr <= most;
        own = {ok ? fr : 0, ok ? pages_of(hd) : 0, ok ? pages_of(kp + fr) : 0, ok ? kp : kRefused};
        have[i] = own.have;
        if constexpr (kEach == kMany) {
            want[i] = own.want;
            kept[i] = own.kept;
            tok[i] = own.tok;
        }
    }
    // Then a run of requests for every thread (one: the same).
    const int each = kEach == kMany ? (a.B + kThreads - 1) / kThreads : 1;
    const int i0 = min(self * each, a.B), i1 = min(i0 + each, a.B);
    if constexpr (kEach == kMany) lds_barrier();
    auto request = [&](int i) { return kEach != kMany ? own : Request{tok[i], have[i], want[i], kept[i]}; };
    int asked[2] = {0, 0}, before_me[2], all_asked[2];
    for (int i = i0; i < i1; ++i) {
        const Request r = request(i);
        asked[0] = add_sat(asked[0], r.tok);
        asked[1] = add_sat(asked[1], max(r.want - r.have, 0));
    }
    prefix_of<kThreads, kEach == kWaves, 2>(asked, asked_sums, before_me, all_asked);
    int t = before_me[0], k = before_me[1];
    const int all_toks = all_asked[0];
    // Granted in request order while pages and token rows last: once one that takes pages is refused
    // for want of pages (or tokens), so is every later one that takes any, so pages taken have no gaps.
    int gives[1] = {0}, took = 0, gv[1], all_gives[1];
    for (int i = i0; i < i1; ++i) {
        Request r = request(i);
        const int tk = max(r.want - r.have, 0);
        tok[i] = t;
        take[i] = k;
        t = add_sat(t, r.tok);
        k = add_sat(k, tk);
        const bool ok = !(r.kept & kRefused) && (tk == 0 || k <= count) && (r.tok == 0 || t <= a.max_tokens);
        if (!ok) {
            r.kept |= kRefused;
            r.want = r.have;
        }
        kept[i] = r.kept;
        want[i] = r.want;
        if constexpr (kEach != kMany) own = r;
        if (ok && tk > 0) took = k;
        gives[0] = add_sat(gives[0], max(r.have - r.want, 0));
    }
    took = wave_top(took);
    if (kEach != kWaves && (tid & (kWave - 1)) == 0) took_sums[tid / kWave] = took;
    prefix_of<kThreads, kEach == kWaves, 1>(gives, given_sums, gv, all_gives);
    for (int i = i0; i < i1; ++i) {
        give[i] = gv[0];
        if constexpr (kEach == kMany) gv[0] = add_sat(gv[0], max(have[i] - want[i], 0));
    }
    // Everything that another workgroup's outputs may overwrite has been read.  Whose turn it is to write
    // those is asked now and looked at last: the answer's way back is not waited for.
    int all_took = took;
    if constexpr (kEach == kWaves) {
        asm volatile("" ::: "memory");     // (alone; a wave's LDS operations run in order)
    } else {
        wait_vm_stores();
        lds_barrier();
        all_took = wave_top((tid & (kWave - 1)) < kThreads / kWave ? took_sums[tid & (kWave - 1)] : 0);
    }
    unsigned before = 0;
    if (tid == 0 && a.grid > 1)
        before = __hip_atomic_fetch_add((unsigned*)a.pool + kPoolTicket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

    int* const ring = a.pool + kPoolRing;
    auto ring_at = [&](int i) {           // entry i of the ring from its head on, i <= P
        const int at = head + i;
        return at >= P ? at - P : at;
    };
    // Tokens: a run of neighbours for every workgroup, whose owners lie between its ends'.
    const int n_tok = min(all_toks, a.max_tokens);
    const int run = (n_tok + a.grid - 1) / a.grid;
    const int x0 = min((int)blockIdx.x * run, n_tok), x1 = min(x0 + run, n_tok);
    if (x0 < x1) {
        int b0 = 0, b1 = a.B - 1;
        if (a.grid > 1) {
            b0 = owner_of(tok, a.B, x0);
            b1 = owner_of(tok, a.B, x1 - 1);
        }
#pragma unroll 4
        for (int x = x0 + tid; x < x1; x += kThreads) {
            const int b = owner(tok, b0, b1, x);
            const int kp = kept[b], pos = (kp & ~kRefused) + (x - tok[b]);
            const int pi = a.shift >= 0 ? pos >> a.shift : pos / a.R;
            if (a.positions) a.positions[x] = pos;
            long long slot = -1;
            if (!(kp & kRefused)) {
                const int* const from = pi < have[b] ? a.table + (size_t)b * a.max_pages + pi
                                                     : ring + ring_at(take[b] + pi - have[b]);
                const int page = *from;
                if (page >= 0 && page < P) slot = (long long)page * a.R + (pos - pi * a.R);
            }
            a.slot_map[x] = slot;
        }
    }
    // Rows behind the last token, so that a step captured for max_tokens stores nothing for them.
    for (int x = n_tok + blockIdx.x * kThreads + tid; x < a.max_tokens; x += a.grid * kThreads) a.slot_map[x] = -1;
    // Pages taken, from the last thread on, and given back, from the middle on: a small call's three
    // kinds of work fall to different waves and wait side by side.
    const int step = a.grid * kThreads, me = blockIdx.x * kThreads + tid;
    for (int x = step - 1 - me; x < all_took; x += step) {
        const int b = owner(take, 0, a.B - 1, x);
        a.table[(size_t)b * a.max_pages + have[b] + x - take[b]] = ring[ring_at(x)];
    }
    // (More given back than the ring has room for means a pool that was not this one's.)
    const int n_give = min(all_gives[0], P - count);
    for (int x = me >= step / 2 ? me - step / 2 : me + step - step / 2; x < n_give; x += step) {
        const int b = owner(give, 0, a.B - 1, x);
        ring[ring_at(count + x)] = a.table[(size_t)b * a.max_pages + want[b] + x - give[b]];
    }
    if (tid == 0) {
        asm volatile("" : "+v"(before));      // not compared, and so waited for, before this
        shared_turn = a.grid == 1 || before == (unsigned)a.grid - 1;
        if (shared_turn && a.grid > 1)
            __hip_atomic_store((unsigned*)a.pool + kPoolTicket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    lds_barrier();
    if (!shared_turn) return;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const int i = self + j * kThreads;
        if (i >= a.B || (kEach == kWaves && tid >= kWave)) break;
        const bool ok = !(kept[i] & kRefused);
        const int fr = (i + 1 < a.B ? tok[i + 1] : all_toks) - tok[i];
        a.held_out[i] = ok ? kp_own[j] + fr : hd_own[j];
        a.lens[i] = ok ? kp_own[j] + fr : kp_own[j];
        a.token_start[i] = tok[i];
    }
    if (tid == 0) {
        a.token_start[a.B] = all_toks;
        int* const next = a.pool_next ? a.pool_next : a.pool;
        next[kPoolHead] = ring_at(all_took);
        next[kPoolCount] = count - all_took + n_give;
    }
}

// Every page free, in order.
__global__ __launch_bounds__(kBlock) void pool_init_kernel(int* pool, int num_pages) {
    const int i = blockIdx.x * kBlock + threadIdx.x;
    if (i < kPoolRing) pool[i] = i == kPoolCount ? num_pages : 0;
    if (i < num_pages) pool[kPoolRing + i] = i;
}

// ------------------------------------------------------------------------------------
// Rows.  Eight lanes hold a row, 8 channels each; a wave takes eight neighbouring tokens of one
// head's K or V, which lie in neighbouring rows of a page (one line of 4-bit rows).  Bound by
// memory: 128 bytes of bf16 and 36 of codes and scale a row.
// ------------------------------------------------------------------------------------
template <int DT> struct Fmt {            // stored bytes of 8 channels
    static constexpr bool kF32 = DT == KVATTN_KV_F32;
    static constexpr bool k4 = DT == KVATTN_KV_INT4 || DT == KVATTN_KV_FP4_E2M1;
    static constexpr bool k8 = DT == KVATTN_KV_INT8 || DT == KVATTN_KV_FP8_E4M3;
    static constexpr bool kCoded = k4 || k8;
    static constexpr int kBytes = kF32 ? 32 : (DT == KVATTN_KV_BF16 ? 16 : (k8 ? 8 : 4));
};

__device__ __forceinline__ void unpack_bf16x8(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = bf16_lo(w[i]);
        x[2 * i + 1] = bf16_hi(w[i]);
    }
}

// A 4-bit row's scale is its largest magnitude times the float nearest 1/7 or 1/6.
template <int DT> constexpr float kScaleOfMax4 = DT == KVATTN_KV_INT4 ? 1.0f / 7.0f : 1.0f / 6.0f;

// Eight 4-bit codes of x / scale; no scale (a row of zeros) and NaN give zero.
template <int DT>
__device__ __forceinline__ uint32_t codes4(const float (&x)[8], float scale) {
    uint32_t w = 0;
    float y[8];
    // x / scale as the division rounds it, in three instructions: the quotient from the rounded reciprocal,
    // its exact remainder, and the correction (Markstein: correct wherever nothing leaves the normal
    // range and the divisor's fraction is not all ones; ties between codes make every bit count).
    const uint32_t bits = __float_as_uint(scale);
    bool plain = bits >= 0x12800000u && bits <= 0x6C800000u && (bits & 0x7FFFFFu) != 0x7FFFFFu;   // 2^-90 .. 2^90
#pragma unroll
    for (int i = 0; i < 8; i += 2) plain = plain && !__builtin_isunordered(x[i], x[i + 1]);
    if (__all(plain)) {
        const float r = 1.0f / scale;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = x[i] * r;
            y[i] = fmaf(fmaf(-q, scale, x[i]), r, q);
            if constexpr (DT == KVATTN_KV_FP4_E2M1) y[i] = copysignf(y[i], x[i]);   // -0: its remainder is +0
        }
    } else {
        const bool live = scale > 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            y[i] = x[i] / scale;
            y[i] = live && y[i] == y[i] ? y[i] : 0.0f;
        }
    }
    if constexpr (DT == KVATTN_KV_FP4_E2M1) {
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.0f, 0);   // nearest, ties to even
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.0f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.0f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.0f, 3);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = (int)fminf(fmaxf(rintf(y[i]), -7.0f), 7.0f) + 8;
            w |= (uint32_t)c << (4 * i);
        }
    }
    return w;
}

template <int DT>
__device__ __forceinline__ void values4(uint32_t w, float (&x)[8]) {
    if constexpr (DT == KVATTN_KV_FP4_E2M1) {
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0);
        const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
        const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2);
        const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
        x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
        x[4] = c[0]; x[5] = c[1]; x[6] = d[0]; x[7] = d[1];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)((int)((w >> (4 * i)) & 15u) - 8);
    }
}

// Where a token's rows lie: by slot (page * R + row of the page), or at the position that the
// append writes (contiguous or paged).
struct RowsArgs {
    uint8_t* kv;
    float* scale;
    void* act;                 // qkv [n][3][NH][64], or the loaded rows [n][2][NH][64]
    const long long* slots;
    const int* cur_len;
    const int* table;
    int lens_per_seq, max_pages, R, num_pages, n, NH, maxT;
    int shift;                 // log2 of R, or -1
};

// A token's place: its rows of part and head are base + (part * part_heads + h) * R.
struct Place {
    size_t base, part_heads;
    int R;
    __device__ __forceinline__ size_t row(int part, int h) const {
        return base + ((size_t)part * part_heads + h) * R;
    }
};

// Whether the token has one, by slot or at the position appended.
template <bool kSlots>
__device__ __forceinline__ bool place_of(const RowsArgs& a, int tok, Place& at) {
    at.part_heads = a.NH;
    at.R = a.R;
    if constexpr (kSlots) {
        const long long slot = a.slots[tok];
        if (slot < 0 || slot >= (long long)a.num_pages * a.R) return false;
        const long long page = a.shift >= 0 ? slot >> a.shift : slot / a.R;
        at.base = (size_t)page * 2 * a.NH * a.R + (size_t)(slot - page * a.R);
        return true;
    }
    const int cl = min(max(a.cur_len[a.lens_per_seq ? tok : 0], 0), a.maxT - 1);
    if (!a.table) {
        at.base = (size_t)tok * a.NH * a.maxT + cl;
        at.part_heads = (size_t)a.n * a.NH;
        at.R = a.maxT;
        return true;
    }
    const int i = cl / a.R, page = a.table[(size_t)tok * a.max_pages + i];
    if (page < 0 || page >= a.num_pages) return false;
    at.base = (size_t)page * 2 * a.NH * a.R + (cl - i * a.R);
    return true;
}

// A wave's work: eight neighbouring tokens of one (part, head).  (Two or four pairs a wave, their loads
// together: 8192 tokens in and out 19.4 and 18.8 us against 19.8, but 160 tokens 5.6 and 6.8 against 4.9.)
struct RowsItem {
    int tok, part, h, c;
};
__device__ __forceinline__ RowsItem rows_item(const RowsArgs& a) {
    const int lane = threadIdx.x & (kWave - 1);
    const int item = blockIdx.x * (kBlock / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int group = item / (2 * a.NH), ph = item - group * 2 * a.NH, part = ph >= a.NH;
    return {group * 8 + (lane >> 3), part, ph - part * a.NH, lane & 7};
}

template <int DT, bool kSlots>
__global__ __launch_bounds__(kBlock) void store_rows_kernel(RowsArgs a) {
    using F = Fmt<DT>;
    const RowsItem it = rows_item(a);
    if (it.tok >= a.n) return;
    const size_t src = (((size_t)it.tok * 3 + 1 + it.part) * a.NH + it.h) * kHd + it.c * 8;
    const uint4* const p = reinterpret_cast<const uint4*>((const uint8_t*)a.act + src * (F::kF32 ? 4 : 2));
    const uint4 x0 = p[0], x1 = F::kF32 ? p[1] : x0;
    Place at;
    if (!place_of<kSlots>(a, it.tok, at)) return;      // the same for a row's eight lanes
    const size_t row = at.row(it.part, it.h);
    uint8_t* const dst = a.kv + (row * 8 + it.c) * F::kBytes;
    if constexpr (!F::kCoded) {
        reinterpret_cast<uint4*>(dst)[0] = x0;
        if constexpr (F::kF32) reinterpret_cast<uint4*>(dst)[1] = x1;
    } else {
        float f[8], amax = 0.0f;
        unpack_bf16x8(x0, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(f[e]));
        amax = row_max<8>(amax);
        const float scale = F::k4 ? amax * kScaleOfMax4<DT> : amax / kW8Limit<F::k8 ? DT : KVATTN_KV_INT8>;
        if (it.c == 0) a.scale[row] = scale;
        if constexpr (F::k4) {
            *reinterpret_cast<uint32_t*>(dst) = codes4<DT>(f, scale);
        } else {
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e / 4] |= (uint32_t)w8_code<DT>(f[e], scale) << (8 * (e % 4));
            *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
        }
    }
}

__device__ __forceinline__ void store16_nt(uint4* p, const uint4& v) {
    typedef unsigned U32x4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(U32x4{v.x, v.y, v.z, v.w}, reinterpret_cast<U32x4*>(p));
}

template <int DT>
__global__ __launch_bounds__(kBlock) void load_rows_kernel(RowsArgs a) {
    using F = Fmt<DT>;
    const RowsItem it = rows_item(a);
    Place at;
    if (it.tok >= a.n || !place_of<true>(a, it.tok, at)) return;
    const size_t row = at.row(it.part, it.h);
    const uint8_t* const src = a.kv + (row * 8 + it.c) * F::kBytes;
    const size_t dst = (((size_t)it.tok * 2 + it.part) * a.NH + it.h) * kHd + it.c * 8;
    uint4* const to = reinterpret_cast<uint4*>((uint8_t*)a.act + dst * (F::kF32 ? 4 : 2));
    if constexpr (!F::kCoded) {
        const uint4* const from = reinterpret_cast<const uint4*>(src);
        const uint4 x0 = from[0], x1 = F::kF32 ? from[1] : x0;
        to[0] = x0;
        if constexpr (F::kF32) to[1] = x1;
    } else {
        const float scale = a.scale[row];
        float x[8];
        if constexpr (F::k4) {
            values4<DT>(*reinterpret_cast<const uint32_t*>(src), x);
        } else {
            const uint2 w = *reinterpret_cast<const uint2*>(src);
            float y[16];
            decode_codes<DT == KVATTN_KV_FP8_E4M3>(make_uint4(w.x, w.y, 0, 0), y);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = y[e];
        }
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            o[e] = f32_to_bf16(x[2 * e] * scale) | (uint32_t)f32_to_bf16(x[2 * e + 1] * scale) << 16;
        // Past the caches: what is loaded is mostly more than they hold.  12 heads of FP4, us without / so: the load alone,
        // 160 tokens 2.4 / 2.4, 4000 6.1 / 5.6, 8192 9.5 / 8.1; stored and loaded, 160 4.8 / 4.8, 8192 18.7 / 17.5; loaded and
        // read by the next kernel, 160 4.4 / 4.6, 1000 6.2 / 6.5, 4000 13.8 / 12.5, 8192 19.5 / 19.8.  The same for
        // what is stored costs 1.4 us.
        store16_nt(to, make_uint4(o[0], o[1], o[2], o[3]));
    }
}

int launch_rows(const void* fn, RowsArgs a, void* stream) {
    a.shift = log2_or(a.R);
    const long long items = (long long)((a.n + 7) / 8) * 2 * a.NH;
    const long long grid = (items + kBlock / kWave - 1) / (kBlock / kWave);
    void* params[] = {&a};
    return hip_status(hipLaunchKernel(fn, dim3((unsigned)grid), dim3(kBlock), params, 0, (hipStream_t)stream));
}

template <template <int> class K>
const void* by_type(int dt) {
    switch (dt) {
        case KVATTN_KV_F32: return K<KVATTN_KV_F32>::fn();
        case KVATTN_KV_BF16: return K<KVATTN_KV_BF16>::fn();
        case KVATTN_KV_INT8: return K<KVATTN_KV_INT8>::fn();
        case KVATTN_KV_FP8_E4M3: return K<KVATTN_KV_FP8_E4M3>::fn();
        case KVATTN_KV_INT4: return K<KVATTN_KV_INT4>::fn();
        case KVATTN_KV_FP4_E2M1: return K<KVATTN_KV_FP4_E2M1>::fn();
        default: return nullptr;
    }
}
template <int DT> struct StoreFn { static const void* fn() { return (const void*)&store_rows_kernel<DT, true>; } };
template <int DT> struct LoadFn { static const void* fn() { return (const void*)&load_rows_kernel<DT>; } };

// Checks shared by paged_store and paged_load, then the launch.
int rows_call(const void* fn, void* act, void* pages, float* scales, int page_rows, int num_pages,
              const long long* slots, int n, int NH, int hs, int dt, void* stream) {
    if (hs != kHd) return KVATTN_ERR_HEAD_DIM;
    if (n < 1 || NH < 1 || page_rows < 1 || page_rows > kMaxT || num_pages < 1) return KVATTN_ERR_SHAPE;
    if (NH > (1 << 24) || (long long)n * NH > (1ll << 27)) return KVATTN_ERR_SHAPE;
    if (!fn) return KVATTN_ERR_DTYPE;
    if (!act || !pages || !slots) return KVATTN_ERR_NULL_POINTER;
    const bool coded = dt != KVATTN_KV_F32 && dt != KVATTN_KV_BF16;
    if (coded && !scales) return KVATTN_ERR_DTYPE;
    if (((uintptr_t)act & 15u) || ((uintptr_t)pages & 15u) || ((uintptr_t)slots & 7u) || ((uintptr_t)scales & 3u))
        return KVATTN_ERR_MISALIGNED;
    RowsArgs a{(uint8_t*)pages, scales, act, slots, nullptr, nullptr, 0, 0, page_rows, num_pages, n, NH, 0, -1};
    return launch_rows(fn, a, stream);
}

}  // namespace

namespace kvattn_internal {
int append4(void* kv, float* scale, const void* qkv, int B, int NH, int maxT, const int* cur_len, int lens_per_seq,
            const int* table, int max_pages, int page_rows, int num_pages, int kv_dtype, void* stream) {
    const void* fn = kv_dtype == KVATTN_KV_INT4 ? (const void*)&store_rows_kernel<KVATTN_KV_INT4, false>
                                                : (const void*)&store_rows_kernel<KVATTN_KV_FP4_E2M1, false>;
    RowsArgs a{(uint8_t*)kv, scale, (void*)qkv, nullptr, cur_len, table, lens_per_seq, max_pages, page_rows, num_pages,
               B, NH, maxT, -1};
    return launch_rows(fn, a, stream);
}
}  // namespace kvattn_internal

extern "C" {

size_t kvattn_paged_pool_bytes(int num_pages) {
    if (num_pages < 1 || num_pages > (1 << 28)) return 0;
    return (size_t)(kPoolRing + num_pages) * sizeof(int);
}

int kvattn_paged_pool_init(int* pool, int num_pages, void* stream) {
    if (num_pages < 1 || num_pages > (1 << 28)) return KVATTN_ERR_SHAPE;
    if (!pool) return KVATTN_ERR_NULL_POINTER;
    if ((uintptr_t)pool & 3u) return KVATTN_ERR_MISALIGNED;
    const int most = num_pages > kPoolRing ? num_pages : kPoolRing;
    void* params[] = {&pool, &num_pages};
    return hip_status(hipLaunchKernel((const void*)&pool_init_kernel, dim3((most + kBlock - 1) / kBlock), dim3(kBlock),
                                      params, 0, (hipStream_t)stream));
}

int kvattn_paged_reserve(int* block_table, int max_pages, int page_rows, int num_pages, int* pool, const int* held,
                         const int* kept, const int* fresh, int B, int max_tokens, int* held_out, int* lens,
                         int* token_start, long long* slot_map, int* positions, int* pool_next, void* stream) {
    if (B < 1 || B > kMaxRequests || max_pages < 1 || page_rows < 1 || num_pages < 1 || num_pages > (1 << 28) ||
        (long long)max_pages * page_rows > kMaxT || max_tokens < 0 || max_tokens > kMostTokens)
        return KVATTN_ERR_SHAPE;
    if (!block_table || !pool || !held || !kept || !fresh || !held_out || !lens || !token_start ||
        (!slot_map && max_tokens > 0))
        return KVATTN_ERR_NULL_POINTER;
    const void* ints[] = {block_table, pool, held, kept, fresh, held_out, lens, token_start, positions, pool_next};
    for (const void* p : ints)
        if ((uintptr_t)p & 3u) return KVATTN_ERR_MISALIGNED;
    if ((uintptr_t)slot_map & 7u) return KVATTN_ERR_MISALIGNED;
    ReserveArgs a{block_table, pool, held, kept, fresh, held_out, lens, token_start, slot_map, positions, pool_next,
                  max_pages, page_rows, num_pages, B, max_tokens, log2_or(page_rows), 1};
    int lds = kRequestInts * B * (int)sizeof(int);
    static_assert(kRequestInts * kMaxRequests * sizeof(int) <= 128 * 1024, "LDS of a CU");
    const bool small = B <= kSmallThreads && max_tokens <= 4 * kSmallThreads;
    const int threads = small ? kSmallThreads : kReserveThreads;
    const bool waves = small && B <= kWave;
    const void* fn = waves                  ? (const void*)&reserve_kernel<kSmallThreads, kWaves>
                     : small                ? (const void*)&reserve_kernel<kSmallThreads, kOne>
                     : B <= kReserveThreads ? (const void*)&reserve_kernel<kReserveThreads, kOne>
                                            : (const void*)&reserve_kernel<kReserveThreads, kMany>;
    if (waves) lds *= kSmallThreads / kWave;
    if (lds > 64 * 1024) {
        const int st = hip_status(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
        if (st != KVATTN_OK) return st;
    }
    const long long blocks = ((long long)max_tokens + kReserveTokens - 1) / kReserveTokens;
    a.grid = (int)(small || blocks < 1 ? 1 : blocks > kReserveMostBlocks ? kReserveMostBlocks : blocks);
    void* params[] = {&a};
    return hip_status(hipLaunchKernel(fn, dim3(a.grid), dim3(threads), params, (size_t)lds, (hipStream_t)stream));
}

int kvattn_paged_store(void* pages, float* page_scales, int page_rows, int num_pages, const long long* slot_map,
                       const void* qkv, int num_tokens, int NH, int hs, int kv_dtype, void* stream) {
    return rows_call(by_type<StoreFn>(kv_dtype), (void*)qkv, pages, page_scales, page_rows, num_pages, slot_map,
                     num_tokens, NH, hs, kv_dtype, stream);
}

int kvattn_paged_load(void* kv, const void* pages, const float* page_scales, int page_rows, int num_pages,
                      const long long* slot_map, int num_tokens, int NH, int hs, int kv_dtype, void* stream) {
    return rows_call(by_type<LoadFn>(kv_dtype), kv, (void*)pages, (float*)page_scales, page_rows, num_pages, slot_map,
                     num_tokens, NH, hs, kv_dtype, stream);
}

}  // extern "C"
