// kv4.hip -- decode attention over a 4-bit KV cache on MI355X (gfx950), for one or several new
// tokens of every sequence.
//
// A row costs 36 bytes, so at the memory's rate a SIMD has about 17 cycles for each: the products go
// to the matrix cores (16x16x32 bf16: codes and q are exact there, sums are float), which leaves the
// vector units the codes' conversion and the softmax.  A wave walks tiles of 64 positions with an
// online softmax.
//   Scores.  The 16 rows of the left operand are 1, 4 or 8 queries, repeated; the columns 16 positions.
//   Of a result, lane 16 g + n holds rows 4 g .. 4 g + 3 of column n, so it takes from the results of
//   the tile's four groups of positions those that no other lane takes for the same query: one
//   position and up to four queries a lane, or two positions and four of eight.  (With queries as columns,
//   one query's softmax was done 16 times over, and that bound the call.)
//   Outputs.  O^T[channel][column] = V^T P^T.  A column is one query's weights in bf16, once their
//   upper half and once the rest (a weight is the sum of the two to 2^-14; one bf16 would round a
//   sharp head's output by 2^-9 before the output's own rounding).  Weights go from positions in lanes
//   to the operand's layout through LDS, and V, which is needed channel-major, through
//   ds_read_b64_tr_b4: lane 16 g + c receives channel c of the 16 rows that group g names.
//
// The FP8-rate matrix instructions would take FP4 codes as they are, but cut small products against
// large ones (2^-14 of the sum of magnitudes, measured), which a score cannot afford.
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
constexpr int kTileBytes = kTile * kRowBytes;
constexpr int kWaveLds = 2 * kTileBytes;   // K (then the weights), V
constexpr int kOutPad = kHd + 4;            // floats from one query's outputs to the next in LDS: other banks
constexpr float kQScale = 0.125f * 1.4426950408889634f;    // 1/sqrt(64) * log2(e)
constexpr float kSlack = 8.0f;
constexpr int kMaxT = 1 << 23;
constexpr int kMaxSegments = 65535;        // the grid's third side
constexpr int kMostWaves = (1 << 26) - 1;  // of a grid: 2^32 threads are too many
// AUTO's shapes.  Up to one head a CU (two where eight queries share a pass, whose heads take longer),
// workgroups of 8 waves, in as many segments as there are CUs; beyond,
// 4 waves, in segments that fill four workgroups a CU, and with ragged lengths past 6144 positions of
// about 32 tiles, so that the longest sequence is not waited for alone.  No segment is shorter than 16
// tiles (a join of segments costs 1 us and more), except where 4 waves split ragged lengths: the long
// sequences' joins are waited for anyway, and the shorter ones end earlier.  us per call, FP4 unless said:
//   12 heads of 1024 positions   8 waves 1 / 4 segments 4.7 / 5.8, 4 waves 1 / 4 segments 5.1 / 5.7
//   12 heads of 8000             8 waves 8 / 4 / 1 segments 7.4 / 8.5 / 15.2, 4 waves 8 segments 7.8
//   192 heads of 4096            8 waves 1 / 2 segments 11.8 / 14.7, 4 waves 4 / 1 segments 13.5 / 13.1
//   288 ragged heads of up to 4096, 8 tokens   8 waves 1 / 2 segments 16.1 / 16.8; 4 waves 3 segments 16.7,
//                                              of 16 tiles at least 17.6, 1 18.3
//   360 ragged heads of up to 2048, 8 tokens   8 waves 13.3, 4 waves 14.1
//   288 ragged heads of up to 4096, 1 token    4 waves 3 segments 14.1, 8 waves 1 segment 14.6
//   480 ragged heads of up to 1024, 4 tokens, INT4   4 waves 9.8, 8 waves 10.4
//   768 ragged heads of up to 8192, INT4       4 waves 4 / 1 segments 43.6 / 46.7, 8 waves 1 segment 46.3
//   768 ragged heads of up to 1024             4 waves 1 / 2 segments 9.2 / 12.1, 8 waves 1 segment 11.0
constexpr int kCUs = 256;
constexpr int kSegTiles = 16, kRaggedSegTiles = 4;
// A cache of more than these bytes is loaded as read only once (its scales are not: their lines are read in
// parts).  64 sequences of 12 heads, us per call, with and without: 8192 ragged INT4 43.8 / 49.1, 4096 INT4
// 39.9 / 45.4, 4096 ragged FP4 25.1 / 26.7; 16 of 4096 FP4 (57 MB) 12.6 / 11.8, 1 of 8000 7.7 / 7.4.
constexpr long long kPositionBytes = 2 * (kRowBytes + 4), kCachedBytes = 128ll << 20;

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
    int line;                  // groups in one line: the number of sequences, else 0
};

// A tile on its way: 16-byte chunks lane and lane + 64 of K and V, and the scales of the kC positions
// that the lane's scores are of (key0 and 32 on).
template <int kC>
struct Raw {
    uint4 k[2], v[2];
    float ks[kC], vs[kC];
    bool there;            // its page is in the pool
};

constexpr size_t kNoPage = ~(size_t)0;

template <int kC, bool kNt>
__device__ __forceinline__ Raw<kC> load_tile(const Args& a, size_t row0, int last, int lane, int key0,
                                              bool there) {
    Raw<kC> r;
    r.there = there;
    const uint8_t* const k = a.kv + row0 * kRowBytes;
    const uint8_t* const v = k + a.v_rows * kRowBytes;
    const float* const s = a.sc + row0;
    // Rows past the last attended one are not read: their lanes read that one again, so that what
    // an unwritten row holds never matters and the end of a page or slot is never passed.
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t at = (uint32_t)min((lane >> 1) + 32 * j, last) * kRowBytes + (lane & 1) * 16;
        r.k[j] = load16<kNt>(k + at);
        r.v[j] = load16<kNt>(v + at);
    }
#pragma unroll
    for (int j = 0; j < kC; ++j) {
        const uint32_t row = min(key0 + 32 * j, last);
        r.ks[j] = s[row];
        r.vs[j] = (s + a.v_rows)[row];
    }
    return r;
}

// Eight 4-bit codes as a matrix-core operand.  FP4: the values, in order.  INT4: 8 + code, which the
// callers take off again: a half byte alone in a byte is an E4M3 number 2^-9 times it, and one
// instruction makes bf16 of two; in the order 0 2 4 6 1 3 5 7.
template <bool kFp4>
__device__ __forceinline__ Bf16x8 operand(uint32_t w) {
    U32x4 d;
    if constexpr (kFp4) {
        d[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0));
        d[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1));
        d[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2));
        d[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3));
    } else {
        const uint32_t even = w & 0x0F0F0F0Fu, odd = (w >> 4) & 0x0F0F0F0Fu;
        d[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, false));
        d[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, true));
        d[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, false));
        d[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, true));
    }
    return __builtin_bit_cast(Bf16x8, d);
}

// The place of code r of eight in operand().
template <bool kFp4>
__device__ __forceinline__ int place(int r) { return kFp4 ? r : ((r & 1) << 2) + (r >> 1); }

// Eight bf16 values in the order of operand()'s.
template <bool kFp4>
__device__ __forceinline__ Bf16x8 in_order(const uint4& w) {
    U32x4 d = {w.x, w.y, w.z, w.w};
    if constexpr (!kFp4) {
        d[0] = (w.x & 0xffffu) | (w.y << 16);
        d[1] = (w.z & 0xffffu) | (w.w << 16);
        d[2] = (w.x >> 16) | (w.y & 0xffff0000u);
        d[3] = (w.z >> 16) | (w.w & 0xffff0000u);
    }
    return __builtin_bit_cast(Bf16x8, d);
}

__device__ __forceinline__ F32x4 mfma(Bf16x8 a, Bf16x8 b, F32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ void put(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get(const float* p) {
    return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// exp2(m - M) with an empty side (m = -inf) weighing nothing.
__device__ __forceinline__ float weight_of(float m, float M) { return m == -INFINITY ? 0.0f : exp2_fast(m - M); }

// The wave's LDS operations run in order, so what its lanes hand one another there needs no barrier;
// this keeps the compiler from moving one lane's reads over another's writes.
__device__ __forceinline__ void lds_order() { asm volatile("" ::: "memory"); }

// Groups of kQ queries in one line, as many as the tokens can fill: sequence b's first is start[b] / kQ + b, and as
// its n tokens make at most start[b + 1] / kQ - start[b] / kQ + 1 of them, no two sequences meet, and all of them end
// before B + num_tokens / kQ.  The last sequence that begins at or before the slot, 64 looked at at once, and
// the group of it (negative: none).
template <int kQ>
__device__ __forceinline__ int sequence_at(const Args& a, int slot, int lane, int& grp) {
    auto first = [&](int b) { return min(max(a.start[b], 0), a.num_tokens) / kQ + b; };
    int b = 0;
    for (int step = a.line > kWave * kWave ? kWave * kWave : a.line > kWave ? kWave : 1;; step /= kWave) {
        const int i = b + lane * step;
        const unsigned long long at = __ballot(i < a.line && first(min(i, a.line - 1)) <= slot);
        b += (63 - __clzll((long long)(at | 1))) * step;
        if (step == 1) break;
    }
    grp = slot - first(b);
    return b;
}

// Keeps a wave's rare branch from becoming selects that every tile runs.
__device__ __forceinline__ void stay_a_branch() { asm volatile(""); }

// kQ: queries of a workgroup (1, 4 or 8); kW: its waves; kNt: codes loaded as read only once.
template <bool kFp4, int kQ, int kW, bool kNt>
__global__ __launch_bounds__(kW * kWave) __attribute__((amdgpu_waves_per_eu(4))) void attend4_kernel(Args a) {
    __shared__ __align__(16) uint8_t lds[kW * kWaveLds];
    __shared__ float red_m[kW][kQ], red_l[kW][kQ];
    __shared__ int is_last;
    static_assert(kQ * kOutPad * 4 <= kWaveLds && kQ * 2 * kTile * 2 <= kTileBytes, "outputs and weights take a tile's place");
    // A lane scores kC positions of a tile for kS of the queries.
    constexpr int kC = kQ <= 4 ? 1 : 2, kS = kQ == 1 ? 1 : 4;

    // Heads lie next to each other in the grid, so that a long sequence's are spread over the XCDs.
    int b = blockIdx.y, grp = a.groups == 1 ? 0 : blockIdx.x / a.NH;
    const int h = blockIdx.x - grp * a.NH, s = blockIdx.z;
    if constexpr (kQ == 8) {
        if (a.line) {
            b = sequence_at<kQ>(a, grp, threadIdx.x & (kWave - 1), grp);
            if (grp < 0) return;
        }
    }
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
    const int q0 = grp * kQ;
    if (q0 >= n) return;
    const int nq = min(kQ, n - q0);
    // Query i of the group attends the first seen0 + i rows.
    const int seen0 = total - n + q0 + 1;
    const int rows = max(seen0 + nq - 1, 0);
    const int tiles = (rows + kTile - 1) / kTile;
    int segs = 1, seg_tiles = tiles;
    if (a.S > 1) {
        seg_tiles = max(a.seg_tiles, (tiles + a.S - 1) / a.S);
        segs = max(1, (tiles + seg_tiles - 1) / seg_tiles);
    }
    if (s >= segs) return;
    const int first = s * seg_tiles, end = min(tiles, first + seg_tiles);

    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, g = lane >> 4;
    const int key0 = 16 * (g / kC) + col, my_q = 4 * (g % kC);   // the first position and query a lane scores
    const int mine = (end - first - wave + kW - 1) / kW;    // tiles of this wave: first + wave + k kW

    // The first rows of this wave's tiles, one a lane, 64 tiles ahead; all ones: no such page.
    size_t starts = 0;
    auto load_starts = [&](int k0) {
        const int pos = (first + wave + (k0 + lane) * kW) * kTile;
        long long id = b;
        int in_page = pos;
        if (a.table) {
            const int page = div_uniform(pos, a.R);
            in_page = pos - page * a.R;
            id = a.table[(size_t)b * a.max_pages + min(page, a.max_pages - 1)];    // (lanes past the last tile)
        }
        const size_t start = (size_t)(id * a.id_mul + h) * a.R + in_page;
        starts = a.table && (id < 0 || id >= a.num_pages) ? kNoPage : start;
    };
    auto start_of = [&](int k) {
        const int lo = __builtin_amdgcn_readlane((int)starts, k & (kWave - 1));
        const int hi = __builtin_amdgcn_readlane((int)(starts >> 32), k & (kWave - 1));
        return ((size_t)(unsigned)hi << 32) | (unsigned)lo;
    };
    // The tile on its way.  Every tile's work asks for the next, behind the last a row again that is there: on a
    // path without, the compiler would count on fewer loads in flight and wait for the newest.  (Two on their
    // way, each waited for alone: 0 to 8 % slower.)
    Raw<kC> raw;
    size_t row0 = 0;
    auto request = [&](int k) {
        if ((k & (kWave - 1)) == 0) load_starts(k);
        const size_t start = start_of(k);
        const int pos = (first + wave + k * kW) * kTile;
        raw.there = k < mine && start != kNoPage;
        if (raw.there) row0 = start;
        raw = load_tile<kC, kNt>(a, row0, k < mine ? min(kTile, rows - pos) - 1 : 0, lane, key0, raw.there);
    };
    // The left operand: row i is query i % kQ (the last one again past it).
    const int qi = min(col % kQ, nq - 1);
    const uint4* const qp = reinterpret_cast<const uint4*>(a.qkv + ((size_t)(t0 + q0 + qi) * 3 * a.NH + h) * kHd + 16 * g);
    const uint4 qw[2] = {qp[0], qp[1]};
    lds_order();
    request(0);
    Bf16x8 qa[2] = {in_order<kFp4>(qw[0]), in_order<kFp4>(qw[1])};
    // Waited for here: left to the loop, their wait would hold up every tile for the next one's loads.
    asm volatile("" : "+v"(qa[0]), "+v"(qa[1]));
    // INT4: the operand's codes are 8 too large, so every score starts at -8 times the sum of q.
    const Bf16x8 minus8 = (Bf16x8)(__bf16)(-8.0f);
    F32x4 s_init = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (!kFp4) s_init = mfma(qa[1], minus8, mfma(qa[0], minus8, s_init));

    uint8_t* const lk = lds + wave * kWaveLds;
    uint8_t* const lv = lk + kTileBytes;
    // Weights [query][upper, rest][place of a position]: with two positions a lane, those are neighbours.
    uint16_t* const lp = reinterpret_cast<uint16_t*>(lk);
    F32x4 acc[4] = {};                     // channels 16 c + 4 g + i of column col: query col % kQ
    // m, alike in a query's lanes, is what the exponents are taken off (off: zero before the first score);
    // limit: the score from which m follows.
    float m[kS], off[kS], limit[kS], l[kS];
#pragma unroll
    for (int i = 0; i < kS; ++i) {
        m[i] = limit[i] = -INFINITY;
        off[i] = l[i] = 0.0f;
    }
    // Column col's weights: query col % kQ, part col / kQ (further columns repeat these).
    const int p_at = ((col & (kQ - 1)) * 2 + ((col / kQ) & 1)) * kTile + 8 * g;
    // The row that this lane names to the transposing read: place 32 (col / 8) + 8 g + place(col % 8).
    const int tr_place = 32 * (col >> 3) + 8 * g + place<kFp4>(col & 7);
    const int tr_row = kC == 1 ? tr_place : (tr_place >> 1) + 32 * (tr_place & 1);

    for (int k = 0; k < mine; ++k) {
        const int pos = (first + wave + k * kW) * kTile;
        const bool there = raw.there;
        float ks[kC], vs[kC];
#pragma unroll
        for (int j = 0; j < kC; ++j) {
            // (Copies that the compiler sees would share the next scales' registers, and be made at the tile's end.)
            asm volatile("v_mov_b32 %0, %2\n\tv_mov_b32 %1, %3" : "=&v"(ks[j]), "=&v"(vs[j]) : "v"(raw.ks[j]), "v"(raw.vs[j]));
            ks[j] *= kQScale;
        }
        lds_order();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            reinterpret_cast<uint4*>(lk)[lane + 64 * j] = raw.k[j];
            reinterpret_cast<uint4*>(lv)[lane + 64 * j] = raw.v[j];
        }
        lds_order();
        request(k + 1);

        uint2 kw[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) kw[t] = *reinterpret_cast<const uint2*>(lk + (16 * t + col) * kRowBytes + 8 * g);
        I32x2 vw[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            vw[c] = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                (__attribute__((address_space(3))) I32x2*)(lv + tr_row * kRowBytes + 8 * c));
        lds_order();
        F32x4 d[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            d[t] = mfma(qa[0], operand<kFp4>(kw[t].x), s_init);
            d[t] = mfma(qa[1], operand<kFp4>(kw[t].y), d[t]);
        }
        // This lane's: group of positions g, or g / 2 and g / 2 + 2.
        float own[kC][kS];
#pragma unroll
        for (int i = 0; i < kS; ++i) {
            if constexpr (kC == 1) {
                const float even = (g & 2) ? d[2][i] : d[0][i], odd = (g & 2) ? d[3][i] : d[1][i];
                own[0][i] = (g & 1) ? odd : even;
            } else {
                own[0][i] = (g & 2) ? d[1][i] : d[0][i];
                own[1][i] = (g & 2) ? d[3][i] : d[2][i];
            }
        }
        // Rows that a query does not see: its later drafts, what is past the last row, a missing page.
        const bool masked = !there || pos + kTile > seen0;
        const int seen = there ? seen0 - pos - key0 + my_q : -kTile;     // query my_q + i sees position key0 + 32 j: seen + i > 32 j
        float sc[kC][kS];
#pragma unroll
        for (int j = 0; j < kC; ++j)
#pragma unroll
            for (int i = 0; i < kS; ++i) {
                sc[j][i] = own[j][i] * ks[j];
            }
        if (masked) {
            stay_a_branch();
#pragma unroll
            for (int j = 0; j < kC; ++j)
#pragma unroll
                for (int i = 0; i < kS; ++i) sc[j][i] = seen + i > 32 * j ? sc[j][i] : -INFINITY;
        }
        bool grows = false;
#pragma unroll
        for (int j = 0; j < kC; ++j)
#pragma unroll
            for (int i = 0; i < kS; ++i) grows |= sc[j][i] > limit[i];
        // Exponents are taken off a maximum that may lag behind by kSlack: weights up to 2^kSlack lose
        // nothing, and after a wave's first tile this is rarely entered.
        if (__any(grows)) {
            float f[kS];
#pragma unroll
            for (int i = 0; i < kS; ++i) {
                float top = sc[0][i];
                if constexpr (kC == 2) top = op_xor32<true>(row_max<16>(fmaxf(top, sc[1][i])));
                else top = wave_max(top);
                const float mn = fmaxf(m[i], top);
                f[i] = weight_of(m[i], mn);
                m[i] = mn;
                off[i] = mn == -INFINITY ? 0.0f : mn;
                limit[i] = mn + kSlack;
                l[i] *= f[i];
            }
            float keep = f[0];
#pragma unroll
            for (int q = 0; q < (kQ == 1 ? 0 : kQ); ++q) {
                const float fq = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f[q % 4]), 16 * (q / 4)));
                keep = (col & (kQ - 1)) == q ? fq : keep;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] *= keep;
        }
#pragma unroll
        for (int j = 0; j < kC; ++j)
#pragma unroll
            for (int i = 0; i < kS; ++i) {
                // Not fused with the product that made the score: the largest one's difference is exact.
#pragma clang fp contract(off)
                const float p = exp2_fast(sc[j][i] - off[i]);
                l[i] += p;
                sc[j][i] = p * vs[j];
            }
        if (masked) {                      // a row that is not seen may have any scale
            stay_a_branch();
#pragma unroll
            for (int j = 0; j < kC; ++j)
#pragma unroll
                for (int i = 0; i < kS; ++i) sc[j][i] = seen + i > 32 * j ? sc[j][i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kS; ++i) {
            uint32_t hi[kC], lo[kC];
#pragma unroll
            for (int j = 0; j < kC; ++j) {
                const float p = sc[j][i];
                hi[j] = __float_as_uint(p);
                lo[j] = __float_as_uint(p - __uint_as_float(hi[j] & 0xffff0000u));
            }
            const int at_q = 2 * (my_q + i) * kTile;
            if constexpr (kC == 1) {
                lp[at_q + lane] = (uint16_t)(hi[0] >> 16);
                lp[at_q + kTile + lane] = (uint16_t)(lo[0] >> 16);
            } else {
                *reinterpret_cast<uint32_t*>(lp + at_q + 2 * key0) = __builtin_amdgcn_perm(hi[1], hi[0], 0x07060302u);
                *reinterpret_cast<uint32_t*>(lp + at_q + kTile + 2 * key0) = __builtin_amdgcn_perm(lo[1], lo[0], 0x07060302u);
            }
        }
        lds_order();
        const Bf16x8 p0 = __builtin_bit_cast(Bf16x8, *reinterpret_cast<const uint4*>(lp + p_at));
        const Bf16x8 p1 = __builtin_bit_cast(Bf16x8, *reinterpret_cast<const uint4*>(lp + p_at + 32));
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if constexpr (!kFp4) {
                acc[c] = mfma(minus8, p0, acc[c]);
                acc[c] = mfma(minus8, p1, acc[c]);
            }
            acc[c] = mfma(operand<kFp4>((uint32_t)vw[c][0]), p0, acc[c]);
            acc[c] = mfma(operand<kFp4>((uint32_t)vw[c][1]), p1, acc[c]);
        }
    }

    // Join the halves of the weights, then the waves.
    lds_order();
    float* const ro = reinterpret_cast<float*>(lk);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            acc[c][i] += kQ == 1 ? dpp<kDppQuadXor1>(acc[c][i])
                                 : (kQ == 4 ? dpp<kDppRowRor4>(acc[c][i]) : dpp<kDppRowRor8>(acc[c][i]));
        if (col < kQ) *reinterpret_cast<F32x4*>(ro + col * kOutPad + 16 * c + 4 * g) = acc[c];
    }
#pragma unroll
    for (int i = 0; i < kS; ++i) {
        l[i] = kC == 2 ? op_xor32<false>(row_sum<16>(l[i])) : wave_sum(l[i]);
        if (col == 0 && g < kC) {
            red_m[wave][my_q + i] = m[i];
            red_l[wave][my_q + i] = l[i];
        }
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
            o += f * reinterpret_cast<const float*>(lds + w * kWaveLds)[qq * kOutPad + ch];
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
        // Eight segments' words on their way at once.
        for (int j0 = 0; j0 < segs; j0 += 8) {
            float mj[8], lj[8], oj[8], top = M;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const size_t slot = slot0 + min(j0 + j, segs - 1);
                mj[j] = get(a.part_max + slot);
                lj[j] = get(a.part_lse + slot);
                oj[j] = get(a.part_out + slot * kHd + ch);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) top = j0 + j < segs ? fmaxf(top, mj[j]) : top;
            const float f0 = weight_of(M, top);
            L *= f0;
            o *= f0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (j0 + j < segs) {
                    const float f = weight_of(mj[j], top);
                    L += f * lj[j];
                    o += f * oj[j];
                }
            }
            M = top;
        }
        a.out[head * kHd + ch] = f32_to_bf16(L == 0.0f ? 0.0f : o / L);
    }
}

template <int kQ, int kW>
const void* kernel_for(bool fp4, bool nt) {
    if (nt) return fp4 ? (const void*)&attend4_kernel<true, kQ, kW, true> : (const void*)&attend4_kernel<false, kQ, kW, true>;
    return fp4 ? (const void*)&attend4_kernel<true, kQ, kW, false> : (const void*)&attend4_kernel<false, kQ, kW, false>;
}
template <int kQ>
const void* kernel_for(bool fp4, int waves, bool nt) {
    return waves == 8 ? kernel_for<kQ, 8>(fp4, nt) : kernel_for<kQ, 4>(fp4, nt);
}

}  // namespace

namespace kvattn_internal {

int plan4(int heads, int queries, int maxT, int len_hint, bool ragged, int S, Plan4& p) {
    const int tiles = ((len_hint >= 0 ? len_hint + 1 : maxT) + kTile - 1) / kTile;
    p.waves = heads <= (queries == 8 ? 2 : 1) * kCUs ? 8 : 4;
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
    p.S = p.waves == 8 ? std::max(1, kCUs / heads) : 4 * kCUs / heads;
    p.S = std::min(p.S, (tiles + kSegTiles - 1) / kSegTiles);
    if (p.waves == 4 && ragged && tiles >= 96) p.S = std::max(p.S, tiles / 32);
    p.S = std::max(1, std::min({p.S, kMaxSegments, kMostWaves / p.waves / heads}));
    // Or ceil(tiles / S), on the device.
    p.seg_tiles = p.waves == 4 && ragged && p.S > 1 ? kRaggedSegTiles : kSegTiles;
    return KVATTN_OK;
}

int attend4(const Attend4& c, bool launch) {
    Plan4 plan;
    // Queries of a workgroup: the fewest that take a sequence's new tokens at once, up to eight.
    const int most_new = c.start ? std::min(c.max_new, c.num_tokens) : 1;
    const int per = most_new == 1 ? 1 : (most_new <= 4 ? 4 : 8);
    // A grid row for every sequence's groups, or all groups in a line where that is shorter: past eight tokens max_new
    // says little about most sequences.  12 heads, us per call, line / rows: 24 ragged sequences of up to 4096,
    // 0 to 8 tokens, max_new 17 / 32 / any 21.0 / 24.6, 20.7 / 20.1, 20.6 / 24.2; 256 of up to 512 16 / 24 / any
    // 24.8 / 26.3, 24.8 / 23.3, 24.6 / 159; 64 of up to 1024, one of them with 200 tokens 14.5 / 20.1.
    const int groups = (most_new + per - 1) / per;
    const long long line = c.B + c.num_tokens / per, each = (long long)c.B * groups;
    const bool in_line = per == 8 && each > line;
    const long long heads = (in_line ? line : each) * c.NH;
    const int st = plan4((int)std::min<long long>(heads, 1 << 30), per, c.maxT, c.len_hint, c.start || c.lens_per_seq,
                         c.S, plan);
    if (st != KVATTN_OK) return st;
    if (c.B > 65535 || heads * plan.S * plan.waves > kMostWaves) return KVATTN_ERR_SHAPE;
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
    a.line = in_line ? c.B : 0;
    a.S = plan.S;
    a.seg_tiles = plan.seg_tiles;
    a.num_tokens = c.num_tokens;
    const bool fp4 = c.kv_dtype == KVATTN_KV_FP4_E2M1;
    long long positions = (long long)c.B * (c.len_hint >= 0 ? c.len_hint + 1 : c.maxT);
    if (c.table) positions = std::min(positions, (long long)c.num_pages * c.page_rows);
    const bool nt = positions > kCachedBytes / kPositionBytes / c.NH;
    const void* fn = per == 1 ? kernel_for<1>(fp4, plan.waves, nt) : per == 4 ? kernel_for<4>(fp4, plan.waves, nt)
                                                                              : kernel_for<8>(fp4, plan.waves, nt);
    void* params[] = {&a};
    const hipError_t e = hipLaunchKernel(fn, in_line ? dim3((unsigned)heads, 1, plan.S) : dim3(c.NH * groups, c.B, plan.S),
                                         dim3(plan.waves * kWave), params, 0, (hipStream_t)c.stream);
    if (e != hipSuccess) {
        set_last_hip_error((int)e);
        return KVATTN_ERR_HIP;
    }
    return KVATTN_OK;
}

}  // namespace kvattn_internal
