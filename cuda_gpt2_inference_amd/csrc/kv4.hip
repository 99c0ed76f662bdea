// kv4.hip -- decode attention over a 4-bit KV cache on MI355X (gfx950), for one or several new
// tokens of every sequence.
//
// A row costs 36 bytes, so at the memory's rate the vector units have about 3.4 instructions for
// each element; the products go to the matrix cores, which leaves the vector units the codes'
// conversion (FP4: one instruction for two values) and the softmax.  A wave walks tiles of 64
// positions with an online softmax:
//   S^T[key][query]  = K Q^T   v_mfma_f32_16x16x32_bf16, codes exact in bf16, q as it is stored
//   O^T[chan][query] = V^T P^T the same; P^T's operand is S^T's result where it lies: lane
//                              16 g + n holds query n at keys 16 t + 4 g + i, and a sum over keys
//                              may take them in any order as long as V's operand does
// V comes row-major and is needed channel-major: tiles pass through the wave's own LDS, and
// ds_read_b64_tr_b4 hands lane 16 g + c channel c of the 16 rows that group g names.
//
// Eight queries share a call to the matrix cores (the drafted tokens of a sequence read the cache
// once).  Each takes two of the 16 columns: a weight p = hi + lo in two bf16 halves, hi in column n
// and lo in column n + 8, so weights keep 14 bits or more where one bf16 would round a sharp head's
// output by 2^-9 before the output's own rounding.  Scores, maxima, sums and outputs are float.
//
// Waves of a workgroup take the tiles of a segment in turn and join through LDS; segments of a
// head join in the workgroup that finishes last (one launch).
#include "kv4.hpp"

#include <math.h>

#include <algorithm>

#include "lanes.hpp"
#include "layout.hpp"

namespace {

using kvattn_internal::Attend4;
using kvattn_internal::Plan4;

typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
typedef int I32x2 __attribute__((ext_vector_type(2)));
typedef float F32x4 __attribute__((ext_vector_type(4)));

constexpr int kHd = 64;
constexpr int kTile = 64;                  // positions of a tile
constexpr int kRowBytes = 32;
constexpr int kGroup = 8;                  // queries of a workgroup
constexpr int kTileBytes = kTile * kRowBytes;
constexpr int kWaveLds = 2 * kTileBytes + 2 * kTile * 4;   // K, V, their scales
constexpr float kQScale = 0.125f * 1.4426950408889634f;    // 1/sqrt(64) * log2(e)
constexpr int kMaxT = 1 << 23;
constexpr int kMaxSegments = 1 << 16;
constexpr int kMostBlocks = 1 << 16;       // AUTO's segments stay longer beyond that many workgroups

struct Args {
    const uint8_t* kv;
    const float* sc;
    const uint16_t* qkv;
    uint16_t* out;
    const int* table;
    const int* start;
    const int* lens;
    float* part_max;
    float* part_lse;
    float* part_out;
    unsigned* counters;
    size_t v_rows;             // rows from a head's K block to its V block
    int id_mul, R;             // a head's block of page (or sequence) id starts at row (id * id_mul + h) * R
    int max_pages, num_pages, lens_per_seq, NH, maxT, groups, S, seg_tiles, num_tokens;
};

// A tile on its way: 16-byte chunks lane and lane + 64 of K and V, row lane's scales.
struct Raw {
    uint4 k[2], v[2];
    float ks, vs;
};

__device__ __forceinline__ Raw load_tile(const Args& a, size_t row0, int last, int lane) {
    Raw r;
    const size_t v0 = row0 + a.v_rows;
    // Rows past the last attended one are not read: their lanes read that one again, so that what
    // an unwritten row holds never matters and the end of a page or slot is never passed.
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t at = (uint32_t)min((lane >> 1) + 32 * j, last) * kRowBytes + (lane & 1) * 16;
        r.k[j] = load16<false>(a.kv + row0 * kRowBytes + at);
        r.v[j] = load16<false>(a.kv + v0 * kRowBytes + at);
    }
    const int row = min(lane, last);
    r.ks = a.sc[row0 + row];
    r.vs = a.sc[v0 + row];
    return r;
}

// Eight 4-bit codes as a matrix-core operand.  FP4: the values, in order (pairs 0 1, 2 3, ...).
// INT4: 24 + code (16 + nibble: the nibble's bits at the top of the mantissa of 16.0), in pairs
// 0 4, 1 5, 2 6, 3 7, which takes two instructions for two values; the callers take the 24 off.
template <bool kFp4>
__device__ __forceinline__ Bf16x8 operand(uint32_t w) {
    U32x4 d;
    if constexpr (kFp4) {
        d[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0));
        d[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1));
        d[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2));
        d[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3));
    } else {
        constexpr uint32_t kMask = 0x00780078u, kBase = 0x41804180u;
        d[0] = ((w << 3) & kMask) | kBase;
        d[1] = ((w >> 1) & kMask) | kBase;
        d[2] = ((w >> 5) & kMask) | kBase;
        d[3] = ((w >> 9) & kMask) | kBase;
    }
    return __builtin_bit_cast(Bf16x8, d);
}

// Eight bf16 values in the order of operand()'s.
template <bool kFp4>
__device__ __forceinline__ Bf16x8 in_order(const uint4& w) {
    U32x4 d = {w.x, w.y, w.z, w.w};
    if constexpr (!kFp4) {
        d[0] = (w.x & 0xffffu) | (w.z << 16);
        d[1] = (w.x >> 16) | (w.z & 0xffff0000u);
        d[2] = (w.y & 0xffffu) | (w.w << 16);
        d[3] = (w.y >> 16) | (w.w & 0xffff0000u);
    }
    return __builtin_bit_cast(Bf16x8, d);
}

__device__ __forceinline__ F32x4 mfma(Bf16x8 a, Bf16x8 b, F32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The upper halves of two floats: both cut to bf16.
__device__ __forceinline__ uint32_t pack_hi(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

__device__ __forceinline__ void put(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get(const float* p) {
    return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// exp2(m - M) with an empty side (m = -inf) weighing nothing.
__device__ __forceinline__ float weight_of(float m, float M) { return m == -INFINITY ? 0.0f : exp2_fast(m - M); }

template <bool kFp4, int kW>
__global__ __launch_bounds__(kW * kWave) void attend4_kernel(Args a) {
    __shared__ __align__(16) uint8_t lds[kW * kWaveLds];
    __shared__ float red_m[kW][kGroup], red_l[kW][kGroup];
    __shared__ int is_last;
    static_assert(kGroup * kHd * 4 <= kWaveLds, "a wave's outputs take its tile's place");

    int x = blockIdx.x;
    const int s = x % a.S;
    x /= a.S;
    const int h = x % a.NH;
    x /= a.NH;
    const int grp = x % a.groups, b = x / a.groups;
    int t0, n, total;
    if (a.start) {
        t0 = min(max(a.start[b], 0), a.num_tokens);
        n = min(max(a.start[b + 1], t0), a.num_tokens) - t0;
        total = min(max(a.lens[a.lens_per_seq ? b : 0], 0), a.maxT);
    } else {
        t0 = b;
        n = 1;
        total = min(max(a.lens[a.lens_per_seq ? b : 0], 0), a.maxT - 1) + 1;
    }
    const int q0 = grp * kGroup;
    if (q0 >= n) return;
    const int nq = min(kGroup, n - q0);
    // Query i of the group attends the first seen0 + i rows.
    const int seen0 = total - n + q0 + 1;
    const int rows = max(seen0 + nq - 1, 0);
    const int tiles = (rows + kTile - 1) / kTile;
    const int seg_tiles = max(a.seg_tiles, (tiles + a.S - 1) / a.S);
    const int segs = max(1, (tiles + seg_tiles - 1) / seg_tiles);
    if (s >= segs) return;
    const int first = s * seg_tiles, end = min(tiles, first + seg_tiles);

    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, g = lane >> 4;
    const int qi = min(col & (kGroup - 1), nq - 1);       // columns past the last query repeat it
    const uint4* qp = reinterpret_cast<const uint4*>(a.qkv + ((size_t)(t0 + q0 + qi) * 3 * a.NH + h) * kHd + 16 * g);
    const uint4 q_lo = qp[0], q_hi = qp[1];

    uint8_t* const lk = lds + wave * kWaveLds;
    uint8_t* const lv = lk + kTileBytes;
    float* const lks = reinterpret_cast<float*>(lk + 2 * kTileBytes);
    float* const lvs = lks + kTile;

    // Pages of this wave's tiles, one a lane, 64 tiles ahead.
    int ids = 0;
    auto load_ids = [&](int k0) {
        const int tile = first + wave + (k0 + lane) * kW;
        ids = b;
        if (a.table) {
            ids = -1;
            if (tile < end) ids = a.table[(size_t)b * a.max_pages + tile * kTile / a.R];
            if (ids >= a.num_pages) ids = -1;
        }
    };
    auto start_tile = [&](int k) {
        const int tile = first + wave + k * kW;
        const int id = max(__builtin_amdgcn_readlane(ids, k & (kWave - 1)), 0);
        const int pos = tile * kTile;
        const size_t row0 = (size_t)((long long)id * a.id_mul + h) * a.R + (a.table ? pos % a.R : pos);
        return load_tile(a, row0, min(kTile, rows - pos) - 1, lane);
    };
    const int mine = (end - first - wave + kW - 1) / kW;    // tiles of this wave
    Raw next;
    if (mine > 0) {
        load_ids(0);
        next = start_tile(0);
    }
    const Bf16x8 qa = in_order<kFp4>(q_lo), qb = in_order<kFp4>(q_hi);
    // INT4: every product is 24 q too large.
    F32x4 s_init = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (!kFp4) {
        float sum = 0.0f;
        const uint32_t w[8] = {q_lo.x, q_lo.y, q_lo.z, q_lo.w, q_hi.x, q_hi.y, q_hi.z, q_hi.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += bf16_lo(w[i]) + bf16_hi(w[i]);
        sum = op_xor32<false>(op_xor16<false>(sum));
        s_init = -24.0f * sum;
    }
    const Bf16x8 minus24 = (Bf16x8)(__bf16)(-24.0f);

    F32x4 acc[4] = {};                     // channels 16 c + 4 g + i of query col
    float m = -INFINITY, l = 0.0f;         // l: this lane's keys alone
    const uint32_t lo_mask = col >= kGroup ? 0xffff0000u : 0u;
    const int tr_row = 16 * (col >> 2) + 4 * g + (col & 3);

    for (int k = 0; k < mine; ++k) {
        const Raw t = next;
        const int pos = (first + wave + k * kW) * kTile;
        const bool there = __builtin_amdgcn_readlane(ids, k & (kWave - 1)) >= 0;
        // The wave's LDS operations run in order, so a tile needs no barrier; the compiler is kept
        // from moving one lane's reads over another's writes.
        asm volatile("" ::: "memory");
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            reinterpret_cast<uint4*>(lk)[lane + 64 * j] = t.k[j];
            reinterpret_cast<uint4*>(lv)[lane + 64 * j] = t.v[j];
        }
        lks[lane] = t.ks * kQScale;
        lvs[lane] = t.vs;
        asm volatile("" ::: "memory");
        if (k + 1 < mine) {
            if (((k + 1) & (kWave - 1)) == 0) load_ids(k + 1);
            next = start_tile(k + 1);
        }

        float sc[16];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
            const uint2 kw = *reinterpret_cast<const uint2*>(lk + (16 * tt + col) * kRowBytes + 8 * g);
            F32x4 d = mfma(operand<kFp4>(kw.x), qa, s_init);
            d = mfma(operand<kFp4>(kw.y), qb, d);
            const F32x4 ks = *reinterpret_cast<const F32x4*>(lks + 16 * tt + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[4 * tt + i] = d[i] * ks[i];
        }
        // Rows that a query does not see: its later drafts, what is past the last row, a missing page.
        const bool masked = !there || pos + kTile > seen0;
        const int seen = there ? seen0 + qi - pos - 4 * g : 0;      // of this lane's keys 16 tt + i
        if (masked) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[e] = 16 * (e >> 2) + (e & 3) < seen ? sc[e] : -INFINITY;
        }
        float top = sc[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, sc[e]);
        top = op_xor32<true>(op_xor16<true>(top));
        const float mn = fmaxf(m, top);
        if (__any(mn != m)) {
            const float keep = weight_of(m, mn);
            l *= keep;
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] *= keep;
            m = mn;
        }
        const float ms = m == -INFINITY ? 0.0f : m;
        float p[16];
        {
            // Not fused with the product that made the score: the largest one's difference is zero.
#pragma clang fp contract(off)
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = exp2_fast(sc[e] - ms);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) l += p[e];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
            const F32x4 vs = *reinterpret_cast<const F32x4*>(lvs + 16 * tt + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) p[4 * tt + i] *= vs[i];
        }
        if (masked) {
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = 16 * (e >> 2) + (e & 3) < seen ? p[e] : 0.0f;
        }
        // hi (columns 0-7) or lo (8-15), both cut: together within 2^-14 of the weight.
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] -= __uint_as_float(__float_as_uint(p[e]) & lo_mask);
        Bf16x8 pw[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            U32x4 d;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                d[j] = kFp4 ? pack_hi(p[8 * u + 2 * j], p[8 * u + 2 * j + 1]) : pack_hi(p[8 * u + j], p[8 * u + 4 + j]);
            pw[u] = __builtin_bit_cast(Bf16x8, d);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const I32x2 vw = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                (__attribute__((address_space(3))) I32x2*)(lv + tr_row * kRowBytes + 8 * c));
            if constexpr (!kFp4) {
                acc[c] = mfma(minus24, pw[0], acc[c]);
                acc[c] = mfma(minus24, pw[1], acc[c]);
            }
            acc[c] = mfma(operand<kFp4>((uint32_t)vw[0]), pw[0], acc[c]);
            acc[c] = mfma(operand<kFp4>((uint32_t)vw[1]), pw[1], acc[c]);
        }
    }

    // Join the halves of the weights, then the waves.
    l = op_xor32<false>(op_xor16<false>(l));
    asm volatile("" ::: "memory");
    float* const ro = reinterpret_cast<float*>(lk);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[c][i] += dpp<kDppRowRor8>(acc[c][i]);
        if (col < kGroup) *reinterpret_cast<F32x4*>(ro + col * kHd + 16 * c + 4 * g) = acc[c];
    }
    if (lane < kGroup) {
        red_m[wave][lane] = m;
        red_l[wave][lane] = l;
    }
    __syncthreads();
    const size_t tok0 = (size_t)t0 + q0;
    for (int e = threadIdx.x; e < nq * kHd; e += kW * kWave) {
        const int qq = e / kHd, ch = e % kHd;
        float M = -INFINITY, L = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < kW; ++w) M = fmaxf(M, red_m[w][qq]);
#pragma unroll
        for (int w = 0; w < kW; ++w) {
            const float f = weight_of(red_m[w][qq], M);
            L += f * red_l[w][qq];
            o += f * reinterpret_cast<const float*>(lds + w * kWaveLds)[e];
        }
        const size_t head = (tok0 + qq) * a.NH + h;
        if (segs == 1) {
            a.out[head * kHd + ch] = f32_to_bf16(L == 0.0f ? 0.0f : o / L);
        } else {
            const size_t slot = head * a.S + s;
            put(a.part_out + slot * kHd + ch, o);
            if (ch == 0) {
                put(a.part_max + slot, M);
                put(a.part_lse + slot, L);
            }
        }
    }
    if (segs == 1) return;

    // The partials are written through to where every XCD reads them; the segment that counts
    // itself last joins them and leaves the counter at zero.
    wait_vm_stores();
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned* const counter = a.counters + tok0 * a.NH + h;
        const unsigned before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        is_last = before == (unsigned)(segs - 1);
        if (is_last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!is_last) return;
    for (int e = threadIdx.x; e < nq * kHd; e += kW * kWave) {
        const int qq = e / kHd, ch = e % kHd;
        const size_t head = (tok0 + qq) * a.NH + h, slot0 = head * a.S;
        float M = -INFINITY, L = 0.0f, o = 0.0f;
        for (int j = 0; j < segs; ++j) M = fmaxf(M, get(a.part_max + slot0 + j));
        for (int j = 0; j < segs; ++j) {
            const float f = weight_of(get(a.part_max + slot0 + j), M);
            L += f * get(a.part_lse + slot0 + j);
            o += f * get(a.part_out + (slot0 + j) * kHd + ch);
        }
        a.out[head * kHd + ch] = f32_to_bf16(L == 0.0f ? 0.0f : o / L);
    }
}

}  // namespace

namespace kvattn_internal {

int plan4(int heads, int maxT, int len_hint, int S, Plan4& p) {
    const int tiles = ((len_hint >= 0 ? len_hint + 1 : maxT) + kTile - 1) / kTile;
    p.waves = 4;
    if (S > 0) {
        if (S > kMaxSegments) return KVATTN_ERR_SPLIT;
        p.S = S;
        p.seg_tiles = 1;
        return KVATTN_OK;
    }
    if (S < 0) {
        if (S < -kMaxT || -S % kTile != 0) return KVATTN_ERR_SPLIT;
        p.seg_tiles = -S / kTile;
        const int most = (maxT + kTile - 1) / kTile;
        p.S = (most + p.seg_tiles - 1) / p.seg_tiles;
        return p.S > kMaxSegments ? KVATTN_ERR_SPLIT : KVATTN_OK;
    }
    p.seg_tiles = 16;
    p.S = (tiles + p.seg_tiles - 1) / p.seg_tiles;
    const int most = kMostBlocks / heads;
    if (p.S > most) p.S = most < 1 ? 1 : most;
    return KVATTN_OK;
}

int attend4(const Attend4& c, bool launch) {
    Plan4 plan;
    const int groups = c.start ? (c.max_new + kGroup - 1) / kGroup : 1;
    const int st = plan4((int)std::min<long long>((long long)c.B * c.NH * groups, 1 << 30), c.maxT, c.len_hint, c.S, plan);
    if (st != KVATTN_OK) return st;
    const long long grid = (long long)c.B * groups * c.NH * plan.S;
    if (grid * plan.waves * kWave > 0xffffffffll) return KVATTN_ERR_SHAPE;
    Args a{};
    if (plan.S > 1) {
        if (!c.ws) return KVATTN_ERR_WORKSPACE;
        if ((uintptr_t)c.ws & 15u) return KVATTN_ERR_MISALIGNED;
        const auto lay = kvattn_layout::ws_layout((long long)c.num_tokens * c.NH, plan.S, c.ws_bytes);
        if (c.ws_bytes == 0 || lay.bytes > c.ws_bytes) return KVATTN_ERR_WORKSPACE;
        uint8_t* const w = (uint8_t*)c.ws;
        a.counters = (unsigned*)(w + lay.counters);
        a.part_max = (float*)(w + lay.part_max);
        a.part_lse = (float*)(w + lay.part_lse);
        a.part_out = (float*)(w + lay.part_out);
    }
    if (!launch) return KVATTN_OK;
    a.kv = (const uint8_t*)c.kv;
    a.sc = c.scale;
    a.qkv = (const uint16_t*)c.qkv;
    a.out = (uint16_t*)c.out;
    a.table = c.table;
    a.start = c.start;
    a.lens = c.lens;
    a.R = c.table ? c.page_rows : c.maxT;
    a.id_mul = c.table ? 2 * c.NH : c.NH;
    a.v_rows = c.table ? (size_t)c.NH * c.page_rows : (size_t)c.B * c.NH * c.maxT;
    a.max_pages = c.max_pages;
    a.num_pages = c.num_pages;
    a.lens_per_seq = c.lens_per_seq;
    a.NH = c.NH;
    a.maxT = c.maxT;
    a.groups = groups;
    a.S = plan.S;
    a.seg_tiles = plan.seg_tiles;
    a.num_tokens = c.num_tokens;
    const bool fp4 = c.kv_dtype == KVATTN_KV_FP4_E2M1;
    const void* fn = fp4 ? (const void*)&attend4_kernel<true, 4> : (const void*)&attend4_kernel<false, 4>;
    void* params[] = {&a};
    const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)grid), dim3(plan.waves * kWave), params, 0,
                                         (hipStream_t)c.stream);
    if (e != hipSuccess) {
        set_last_hip_error((int)e);
        return KVATTN_ERR_HIP;
    }
    return KVATTN_OK;
}

}  // namespace kvattn_internal
