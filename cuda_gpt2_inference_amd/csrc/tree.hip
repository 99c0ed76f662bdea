// tree.hip -- attention of a tree of drafted tokens over a paged KV cache on MI355X (gfx950), for every cache
// type, and the trees' masks.
//
// A sequence's n new tokens are nodes of a tree; their K and V rows are the cache's last n.  Token i attends the
// prefix before them and the new tokens whose bits its mask has (itself and its ancestors).  A workgroup serves 16 of a
// tree's tokens, the columns of a product; those of larger trees run side by side, so that what one loads the others
// find in the caches.  (Two or four groups of 16 in one workgroup take registers that other workgroups hide latency
// with: BF16, 26 tokens over 1000 positions 9.6 us in place of 7.6, INT4 64 x 64 tokens 43.4 and 41.0, BF16 16 x 64 over
// 8192 46.0 and 46.6.  One behind the other on one XCD they share its L2, which then reads the cache once, but a long
// sequence's wait for one another: BF16 16 x 64 45.7 us of 48.2, INT4 64 x 64 47.6 of 41.1.  All on one state, whose cache
// rows the Infinity Cache holds, INT4's in weights of one float16; in turn with others BF16 16 x 64 takes 60.)
//
// Both products go to the matrix cores, scores as S^T = K Q^T and outputs as O^T = V^T P^T.  Of S^T lane
// 16 g + c holds positions 16 t + 4 g .. + 3 of query c.  That makes everything the softmax does (maximum, sum,
// rescaling of the outputs, which are channels of query c in the same lane) a lane's own affair; only a new
// maximum crosses lanes.  And the weights are the second product's operand where they are: the order of positions
// in a sum is free, so a lane's eight places of step s are positions 32 s + 4 g .. + 3 and 32 s + 16 + 4 g .. + 3,
// and V, which is needed channel-major, is read from LDS by the transposing reads (ds_read_b64_tr_b16, b8, b4)
// in that order.
//   Types.  BF16 rows are operands as they are; 8-bit and 4-bit codes are exact in bf16, and their scales go to
//   the scores and the weights in float.  FP32 rows take 16x16x4 float products.  Weights (over codes times their rows'
//   scales) are two bf16 halves, upper and rest, 2^-14 of each, whatever the others are: one half alone would round a sharp
//   head's output (2^-8) twice.  (One float16 is less work, but scales need all of a float's exponents: it takes a unit
//   that the rows share, and rows whose scales lie far below another's, which may not even be attended, were lost in it.)
//   Masks.  Only tiles that reach the new tokens look at any.  There a value that one query must not see may be
//   infinite or NaN, which a weight of zero does not take out of a product: such a tile, found by looking at its V
//   rows, has its outputs summed on the vector units, position by position.
//
// Waves of a workgroup take tiles in turn and join through LDS; segments of a head join in the workgroup that
// finishes last (one launch).
#include "tree.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "lanes.hpp"
#include "layout.hpp"
#include "matrix.hpp"

namespace {

using kvattn_internal::AttendTree;
using kvattn_internal::kMaxMaskWords;
using kvattn_internal::kMaxTree;

constexpr int kHd = 64;
constexpr int kSeg = 64;                   // positions that segments are counted in
constexpr int kQ = 16;                     // queries of a group: columns of a product
constexpr int kOutPad = kHd + 4;           // floats from one query's outputs to the next in LDS: other banks
constexpr float kQScale = 0.125f * 1.4426950408889634f;    // 1/sqrt(64) * log2(e)
constexpr float kSlack = 8.0f;
constexpr int kMaxSegments = 65535;        // the grid's third side
constexpr int kMostWaves = (1 << 26) - 1;  // of a grid: 2^32 threads are too many
constexpr int kCUs = 256, kFewHeads = 32;

template <int DT> struct Kv {
    static constexpr bool kF32 = DT == KVATTN_KV_F32;
    static constexpr bool kBf16 = DT == KVATTN_KV_BF16;
    static constexpr bool k8 = DT == KVATTN_KV_INT8 || DT == KVATTN_KV_FP8_E4M3;
    static constexpr bool kFp8 = DT == KVATTN_KV_FP8_E4M3;
    static constexpr bool k4 = DT == KVATTN_KV_INT4 || DT == KVATTN_KV_FP4_E2M1;
    static constexpr bool kFp4 = DT == KVATTN_KV_FP4_E2M1;
    static constexpr bool kInt4 = DT == KVATTN_KV_INT4;
    static constexpr bool kCoded = k8 || k4;
    static constexpr int kRow = kF32 ? 256 : kBf16 ? 128 : k8 ? 64 : 32;      // bytes
    static constexpr int kChunks = kRow / 16;
    static constexpr int kPos = kF32 ? 16 : kBf16 ? 32 : 64;                  // positions of a wave's tile: up to 8 KB
    static constexpr bool kMayBeInfinite = kF32 || kBf16 || kFp8;             // (FP8 has a NaN)
    // Where chunk c of a row lies among the row's chunks in LDS, so that the rows that are read together
    // lie in different banks.
    __device__ static __forceinline__ int chunk_at(int row, int c) {
        if constexpr (kF32) return c ^ (row & 15);
        if constexpr (kBf16) return c ^ (row & 7);
        if constexpr (k8) return c ^ ((row >> 2) & 3);
        return c;
    }
};

struct TreeArgs {
    const uint8_t* kv;
    const float* sc;
    const uint8_t* qkv;
    uint8_t* out;
    const int* table;
    const int* start;
    const int* lens;
    const unsigned long long* masks;
    float* part_max;
    float* part_lse;
    float* part_out;
    unsigned* counters;
    size_t v_rows;             // rows from a head's K block to its V block
    int R, max_pages, num_pages, NH, maxT, words, S, seg_tiles, num_tokens;
};

constexpr size_t kNoPage = ~(size_t)0;

// One element of a V row in LDS as a float (without its scale).
template <int DT>
__device__ __forceinline__ float element(const uint8_t* lv, int row, int ch) {
    using T = Kv<DT>;
    if constexpr (T::kF32) {
        return *reinterpret_cast<const float*>(lv + row * T::kRow + 16 * T::chunk_at(row, ch / 4) + 4 * (ch % 4));
    } else if constexpr (T::kBf16) {
        return bf16_to_f32(*reinterpret_cast<const uint16_t*>(lv + row * T::kRow + 16 * T::chunk_at(row, ch / 8) + 2 * (ch % 8)));
    } else {
        const int c = lv[row * T::kRow + 16 * T::chunk_at(row, ch / 16) + ch % 16];
        return __builtin_amdgcn_cvt_pk_f32_fp8(c, false)[0];
    }
}

// Whether any of a chunk's elements is infinite or NaN.
template <int DT>
__device__ __forceinline__ bool not_finite(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (Kv<DT>::kF32) {
            bad |= (w[i] & 0x7f800000u) == 0x7f800000u;
        } else if constexpr (Kv<DT>::kBf16) {
            bad |= (w[i] & 0x7f800000u) == 0x7f800000u || (w[i] & 0x7f80u) == 0x7f80u;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) bad |= ((w[i] >> (8 * k)) & 0x7fu) == 0x7fu;
        }
    }
    return bad;
}

// Four neighbouring outputs; a query that attends nothing has none.
template <bool kF32>
__device__ __forceinline__ void store_out(uint8_t* out, size_t at, float L, F32x4 o) {
    o = L == 0.0f ? F32x4{0.0f, 0.0f, 0.0f, 0.0f} : o / L;
    if constexpr (kF32) {
        *reinterpret_cast<F32x4*>(out + at * 4) = o;
    } else {
        *reinterpret_cast<uint2*>(out + at * 2) =
            make_uint2(f32_to_bf16(o[0]) | (uint32_t)f32_to_bf16(o[1]) << 16, f32_to_bf16(o[2]) | (uint32_t)f32_to_bf16(o[3]) << 16);
    }
}

// kW: waves of a workgroup.
template <int DT, int kW>
__global__ __launch_bounds__(kW * kWave) __attribute__((amdgpu_waves_per_eu(3))) void tree_kernel(TreeArgs a) {
    using T = Kv<DT>;
    constexpr int kPos = T::kPos, kT = kPos / 16;              // positions of a wave's tile, groups of 16 of them
    constexpr int kTileBytes = kPos * T::kRow;
    constexpr int kLoads = kTileBytes / 1024;                  // 16-byte chunks a lane, of K and of V
    constexpr int kScales = T::kCoded ? 2 * kPos * 4 : 0;
    constexpr int kWaveLds = std::max(2 * kTileBytes + kScales, kQ * kOutPad * 4);
    static_assert(kPos == 64 || !T::kCoded, "a lane holds one position's scales");
    static_assert(kTileBytes % 1024 == 0 && kWaveLds % 16 == 0, "whole loads");
    __shared__ __align__(16) uint8_t lds[kW * kWaveLds];
    __shared__ float red_m[kW][kQ], red_l[kW][kQ];
    __shared__ int is_last;

    const int b = blockIdx.y, grp = blockIdx.x / a.NH, h = blockIdx.x - grp * a.NH, s = blockIdx.z;
    const int t0 = min(max(a.start[b], 0), a.num_tokens);
    const int n = min(max(a.start[b + 1], t0), a.num_tokens) - t0;
    const int total = min(max(a.lens[b], 0), a.maxT);
    const int q0 = grp * kQ;
    if (q0 >= n) return;
    const int nq = min(kQ, n - q0);
    const int base = total - n;                                // position of new token 0
    const int seg_count = (total + kSeg - 1) / kSeg;
    int segs = 1, seg_tiles = seg_count;
    if (a.S > 1) {
        seg_tiles = max(a.seg_tiles, (seg_count + a.S - 1) / a.S);
        segs = max(1, (seg_count + seg_tiles - 1) / seg_tiles);
    }
    if (s >= segs) return;
    const int pos_lo = s * seg_tiles * kSeg, pos_hi = min(total, pos_lo + seg_tiles * kSeg);

    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, g = lane >> 4;
    const int tiles = (pos_hi - pos_lo + kPos - 1) / kPos;
    const int mine = (tiles - wave + kW - 1) / kW;             // tiles of this wave: wave + k kW
    auto pos_of = [&](int k) { return pos_lo + (wave + k * kW) * kPos; };

    // The first rows of this wave's tiles, one a lane, 64 tiles ahead; all ones: no such page.
    size_t starts = 0;
    auto load_starts = [&](int k0) {
        const int pos = pos_of(k0 + lane);
        const int page = div_uniform(pos, a.R);
        const long long id = a.table[(size_t)b * a.max_pages + min(page, a.max_pages - 1)];    // (lanes past the last tile)
        starts = id < 0 || id >= a.num_pages ? kNoPage : (size_t)(id * 2 * a.NH + h) * a.R + (pos - page * a.R);
    };
    auto start_of = [&](int k) {
        const int lo = __builtin_amdgcn_readlane((int)starts, k & (kWave - 1));
        const int hi = __builtin_amdgcn_readlane((int)(starts >> 32), k & (kWave - 1));
        return ((size_t)(unsigned)hi << 32) | (unsigned)lo;
    };
    // The tile on its way: chunks lane, lane + 64, ... of K and V, and the scales of position `lane`.  Rows past the
    // last position are not read: their lanes read that one again.
    uint4 rk[kLoads], rv[kLoads];
    float rks = 0.0f, rvs = 0.0f;
    bool there = false;
    size_t row0 = 0;
    auto request = [&](int k) {
        if ((k & (kWave - 1)) == 0) load_starts(k);
        const size_t start = start_of(k);
        there = k < mine && start != kNoPage;
        if (there) row0 = start;
        const int last = k < mine ? min(kPos, total - pos_of(k)) - 1 : 0;
        const uint8_t* const kp = a.kv + row0 * T::kRow;
        const uint8_t* const vp = kp + a.v_rows * T::kRow;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int c = lane + kWave * j;
            const uint32_t at = (uint32_t)min(c / T::kChunks, last) * T::kRow + (c % T::kChunks) * 16;
            rk[j] = load16<false>(kp + at);
            rv[j] = load16<false>(vp + at);
        }
        if constexpr (T::kCoded) {
            const float* const sp = a.sc + row0 + min(lane, last);
            rks = sp[0];
            rvs = sp[a.v_rows];
        }
    };

    // Queries: column c is query c (the last one again past it), in the order of K's operands.
    constexpr int kQu = T::kF32 ? 4 : 2;                       // 16-byte pieces of a lane
    const size_t my_tok = (size_t)t0 + q0 + min(col, nq - 1);
    const unsigned long long* const my_mask = a.masks + my_tok * a.words;
    uint4 qw[kQu];
#pragma unroll
    for (int u = 0; u < kQu; ++u)
        qw[u] = *reinterpret_cast<const uint4*>(a.qkv + (my_tok * 3 * a.NH + h) * kHd * (T::kF32 ? 4 : 2) +
                                                (T::kCoded ? 32 * g + 16 * u : 64 * u + 16 * g));
    if (mine > 0) request(0);
    const unsigned long long mask0 = my_mask[0];
    Bf16x8 qa[2];
    float q_init = 0.0f;                   // INT4: the operand's codes are 8 too large, so a score starts at -8 sum q
    if constexpr (!T::kF32) {
#pragma unroll
        for (int u = 0; u < 2; ++u) qa[u] = T::kInt4 ? in_order<false>(qw[u]) : __builtin_bit_cast(Bf16x8, qw[u]);
        if constexpr (T::kInt4) {
            const Bf16x8 minus8 = (Bf16x8)(__bf16)(-8.0f);
            const F32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
            q_init = mfma(minus8, qa[1], mfma(minus8, qa[0], zero))[0];
        }
    }

    uint8_t* const lk = lds + wave * kWaveLds;
    uint8_t* const lv = lk + kTileBytes;
    float* const ls = reinterpret_cast<float*>(lv + kTileBytes);
    F32x4 acc[4] = {};                     // channels 16 c + 4 g + i of query col
    F32x4 acc8 = {};                       // INT4: 8 sum of the weights, taken off at the end
    // off: what the exponents are taken off (zero before the first score); limit: the score from which m follows.
    float m = -INFINITY, limit = -INFINITY, off = 0.0f, l = 0.0f;

    for (int k = 0; k < mine; ++k) {
        const int pos = pos_of(k);
        const bool here = there;
        const bool tail = pos + kPos > base;   // some positions are new tokens', or past the last
        bool bad = false;
        if constexpr (T::kMayBeInfinite) {
            if (tail) {
                stay_a_branch();
                bool mine_bad = false;
#pragma unroll
                for (int j = 0; j < kLoads; ++j) mine_bad |= not_finite<DT>(rv[j]);
                bad = __any(mine_bad);
            }
        }
        lds_order();
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int c = lane + kWave * j, row = c / T::kChunks;
            const int at = row * T::kRow + 16 * T::chunk_at(row, c % T::kChunks);
            *reinterpret_cast<uint4*>(lk + at) = rk[j];
            *reinterpret_cast<uint4*>(lv + at) = rv[j];
        }
        if constexpr (T::kCoded) {
            ls[lane] = rks * kQScale;
            ls[kPos + lane] = rvs;
        }
        lds_order();
        if (k + 1 < mine) request(k + 1);
        if (!here) continue;                   // its page is not in the pool

        // Positions that the query sees, one bit each.
        unsigned long long vis = ~0ull;
        if (tail) {
            stay_a_branch();
            const int d = pos - base, w0 = d >> 6, sh = d & 63;      // (d may be negative: words before the first are the prefix)
            const int left = total - pos;
            auto word = [&](int w) { return w < 0 ? ~0ull : w == 0 ? mask0 : w < a.words ? my_mask[w] : 0ull; };
            vis = word(w0) >> sh;
            if (sh) vis |= word(w0 + 1) << (64 - sh);
            vis &= left >= 64 ? ~0ull : (1ull << left) - 1;
        }
        const unsigned long long seen = vis >> (4 * g);

        // Scores.
        F32x4 p[kT];
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            const int row = 16 * t + col;
            p[t] = F32x4{q_init, q_init, q_init, q_init};
            if constexpr (T::kF32) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const U32x4 kf = *reinterpret_cast<const U32x4*>(lk + row * T::kRow + 16 * T::chunk_at(row, 4 * j + g));
                    const uint32_t qv[4] = {qw[j].x, qw[j].y, qw[j].z, qw[j].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        p[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[e]), __uint_as_float(qv[e]), p[t], 0, 0, 0);
                }
            } else {
                Bf16x8 ka[2];
                if constexpr (T::kBf16) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        ka[u] = *reinterpret_cast<const Bf16x8*>(lk + row * T::kRow + 16 * T::chunk_at(row, 4 * u + g));
                } else if constexpr (T::k8) {
                    codes_to_bf16<T::kFp8>(*reinterpret_cast<const U32x4*>(lk + row * T::kRow + 16 * T::chunk_at(row, g)), ka);
                } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(lk + row * T::kRow + 8 * g);
                    ka[0] = operand<T::kFp4>(w.x);
                    ka[1] = operand<T::kFp4>(w.y);
                }
                p[t] = mfma(ka[0], qa[0], p[t]);
                p[t] = mfma(ka[1], qa[1], p[t]);
            }
            if constexpr (T::kCoded) p[t] *= *reinterpret_cast<const F32x4*>(ls + 16 * t + 4 * g);
            else p[t] *= kQScale;
        }
        if (tail) {
            stay_a_branch();
#pragma unroll
            for (int t = 0; t < kT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[t][e] = (seen >> (16 * t + e)) & 1 ? p[t][e] : -INFINITY;
        }
        float top = p[0][0];
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, p[t][e]);
        // Exponents are taken off a maximum that may lag behind by kSlack: weights up to 2^kSlack lose
        // nothing, and after a wave's first tile this is rarely entered.
        if (__any(top > limit)) {
            top = op_xor32<true>(op_xor16<true>(top));
            const float mn = fmaxf(m, top), f = weight_of(m, mn);
            m = mn;
            off = mn == -INFINITY ? 0.0f : mn;
            limit = mn + kSlack;
            l *= f;
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] *= f;
            if constexpr (T::kInt4) acc8 *= f;
        }
        // Weights, over codes times their rows' scales.
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            F32x4 vs = {1.0f, 1.0f, 1.0f, 1.0f};
            if constexpr (T::kCoded) vs = *reinterpret_cast<const F32x4*>(ls + kPos + 16 * t + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // Not fused with the product that made the score: the largest one's difference is exact.
#pragma clang fp contract(off)
                const float w = exp2_fast(p[t][e] - off);
                l += w;
                p[t][e] = T::kCoded ? w * vs[e] : w;
            }
        }
        if (T::kCoded && tail) {               // a row that is not seen may have any scale
            stay_a_branch();
#pragma unroll
            for (int t = 0; t < kT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) p[t][e] = (seen >> (16 * t + e)) & 1 ? p[t][e] : 0.0f;
        }
        if (T::kMayBeInfinite && bad) {
            stay_a_branch();
            // The weights [query][position] in K's place, then position by position.
            static_assert(kQ * kPos * 4 <= kTileBytes || !T::kMayBeInfinite, "weights take K's place");
            float* const lp = reinterpret_cast<float*>(lk) + col * kPos;
            lds_order();
#pragma unroll
            for (int t = 0; t < kT; ++t) *reinterpret_cast<F32x4*>(lp + 16 * t + 4 * g) = p[t];
            lds_order();
#pragma unroll 1
            for (int row = 0; row < kPos; ++row) {
                const float w = lp[row];
                if ((vis >> row) & 1) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            acc[c][x] += w * element<T::kMayBeInfinite ? DT : KVATTN_KV_F32>(lv, row, 16 * c + 4 * g + x);
                }
            }
            lds_order();
            continue;
        }
        // Outputs.  V's operands, transposed: step u's places of channels 16 c + col.
        if constexpr (T::kF32) {
#pragma unroll
            for (int t = 0; t < kT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = 16 * t + 4 * g + e;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float v = *reinterpret_cast<const float*>(lv + row * T::kRow + 16 * T::chunk_at(row, 4 * c + (col >> 2)) +
                                                                        4 * (col & 3));
                        acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[t][e], acc[c], 0, 0, 0);
                    }
                }
        } else {
            // Step u's weights in two halves.
            constexpr int kU = kPos / 32;
            Bf16x8 hi[kU], lo[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                U32x4 h, l;
#pragma unroll
                for (int j = 0; j < 4; ++j) {                  // places 2 j and 2 j + 1
                    const float p0 = p[2 * u + j / 2][2 * (j % 2)], p1 = p[2 * u + j / 2][2 * (j % 2) + 1];
                    const uint32_t b0 = __float_as_uint(p0), b1 = __float_as_uint(p1);
                    h[j] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
                    const float r0 = p0 - __uint_as_float(b0 & 0xffff0000u), r1 = p1 - __uint_as_float(b1 & 0xffff0000u);
                    l[j] = __builtin_amdgcn_perm(__float_as_uint(r1), __float_as_uint(r0), 0x07060302u);
                }
                hi[u] = __builtin_bit_cast(Bf16x8, h);
                lo[u] = __builtin_bit_cast(Bf16x8, l);
                if constexpr (T::kInt4) {
                    acc8 = mfma((Bf16x8)(__bf16)8.0f, hi[u], acc8);
                    acc8 = mfma((Bf16x8)(__bf16)8.0f, lo[u], acc8);
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                Bf16x8 va[2];
                if constexpr (T::kBf16) {
                    typedef short S16x4 __attribute__((ext_vector_type(4)));
                    S16x4 part[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int row = 16 * e + 4 * g + (col >> 2);
                        part[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) S16x4*)(lv + row * T::kRow +
                                16 * T::chunk_at(row, 2 * c + ((col >> 1) & 1)) + 8 * (col & 1)));
                    }
                    va[0] = __builtin_bit_cast(Bf16x8, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
                } else if constexpr (T::k8) {
                    I32x2 part[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int e = col >> 1, row = 32 * u + 16 * (e >> 2) + 4 * g + (e & 3);
                        part[u] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                            (__attribute__((address_space(3))) I32x2*)(lv + row * T::kRow + 16 * T::chunk_at(row, c) + 8 * (col & 1)));
                    }
                    codes_to_bf16<T::kFp8>(U32x4{(uint32_t)part[0][0], (uint32_t)part[0][1], (uint32_t)part[1][0], (uint32_t)part[1][1]}, va);
                } else {
                    const int e = place<T::kFp4>(col & 7), row = 32 * (col >> 3) + 16 * (e >> 2) + 4 * g + (e & 3);
                    const I32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                        (__attribute__((address_space(3))) I32x2*)(lv + row * T::kRow + 8 * c));
                    va[0] = operand<T::kFp4>((uint32_t)v[0]);
                    va[1] = operand<T::kFp4>((uint32_t)v[1]);
                }
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    acc[c] = mfma(va[u], hi[u], acc[c]);
                    acc[c] = mfma(va[u], lo[u], acc[c]);
                }
            }
        }
        lds_order();
    }

    // Join the waves.
    constexpr int kVec = 4, kItems = kHd / kVec;
    const size_t tok0 = (size_t)t0 + q0;
    float* const ro = reinterpret_cast<float*>(lk);
    lds_order();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if constexpr (T::kInt4) acc[c] -= acc8;
        *reinterpret_cast<F32x4*>(ro + col * kOutPad + 16 * c + 4 * g) = acc[c];
    }
    const float sum = op_xor32<false>(op_xor16<false>(l));
    if (g == 0) {
        red_m[wave][col] = m;
        red_l[wave][col] = sum;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nq * kItems; e += kW * kWave) {
        const int qq = e / kItems, ch = e % kItems * kVec;
        float M = -INFINITY, L = 0.0f;
        F32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kW; ++w) M = fmaxf(M, red_m[w][qq]);
#pragma unroll
        for (int w = 0; w < kW; ++w) {
            const float f = weight_of(red_m[w][qq], M);
            L += f * red_l[w][qq];
            o += f * *reinterpret_cast<const F32x4*>(lds + w * kWaveLds + (qq * kOutPad + ch) * 4);
        }
        const size_t head = (tok0 + qq) * a.NH + h;
        if (segs == 1) {
            store_out<T::kF32>(a.out, head * kHd + ch, L, o);
        } else {
            const size_t slot = head * a.S + s;
            put4(a.part_out + slot * kHd + ch, o);
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
    // What an earlier call left of the partials in this XCD's caches is dropped; plain loads of 16 bytes then.
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    for (int e = threadIdx.x; e < nq * kItems; e += kW * kWave) {
        const int qq = e / kItems, ch = e % kItems * kVec;
        const size_t head = (tok0 + qq) * a.NH + h, slot0 = head * a.S;
        float M = -INFINITY, L = 0.0f;
        F32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        // Eight segments' words on their way at once.
        for (int j0 = 0; j0 < segs; j0 += 8) {
            float mj[8], lj[8], top = M;
            F32x4 oj[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const size_t slot = slot0 + min(j0 + j, segs - 1);
                mj[j] = a.part_max[slot];
                lj[j] = a.part_lse[slot];
                oj[j] = *reinterpret_cast<const F32x4*>(a.part_out + slot * kHd + ch);
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
        store_out<T::kF32>(a.out, head * kHd + ch, L, o);
    }
}

template <int DT>
const void* kernel_for(int waves) {
    return waves == 8 ? (const void*)&tree_kernel<DT, 8> : (const void*)&tree_kernel<DT, 4>;
}

// ------------------------------------------------------------------------------------
// Masks and positions from every token's parent.
// ------------------------------------------------------------------------------------
struct MaskArgs {
    unsigned long long* masks;
    int* positions;
    const int* parents;
    const int* start;
    const int* lens;
    int B, num_tokens, words;
};

// One workgroup a sequence, one token a thread.  A parent's index is below its child's, so the way up ends, and
// meets a mask's words from the last to the first.
__global__ __launch_bounds__(kMaxTree) void tree_masks_kernel(MaskArgs a) {
    __shared__ int parent[kMaxTree];
    const int b = blockIdx.x, i = threadIdx.x;
    const int t0 = min(max(a.start[b], 0), a.num_tokens);
    const int n = min(max(a.start[b + 1], t0), a.num_tokens) - t0;
    const int most = min(n, 64 * a.words);
    if (i < most) {
        const int p = a.parents[t0 + i];
        parent[i] = p >= 0 && p < i ? p : -1;
    }
    __syncthreads();
    for (int t = i; t < n; t += kMaxTree) {
        unsigned long long* const out = a.masks + (size_t)(t0 + t) * a.words;
        int depth = 0;
        if (t < most) {
            int w = a.words - 1;
            unsigned long long bits = 0;
            for (int at = t; at >= 0; at = parent[at]) {
                for (; w > at >> 6; --w) {
                    out[w] = bits;
                    bits = 0;
                }
                bits |= 1ull << (at & 63);
                ++depth;
            }
            for (; w >= 0; --w) {
                out[w] = bits;
                bits = 0;
            }
            --depth;
        } else {                               // no bit for it
            for (int w = 0; w < a.words; ++w) out[w] = 0;
        }
        if (a.positions) a.positions[t0 + t] = max(a.lens[b] - n + depth, 0);
    }
}

int hip_status(hipError_t e) {
    if (e == hipSuccess) return KVATTN_OK;
    kvattn_internal::set_last_hip_error((int)e);
    return KVATTN_ERR_HIP;
}

}  // namespace

namespace kvattn_internal {

int attend_tree(const AttendTree& c) {
    const int most_new = std::min(c.max_new, c.num_tokens);
    const int passes = (most_new + kQ - 1) / kQ;
    const long long heads = (long long)c.B * c.NH * passes;
    // Workgroups of 8 waves where there are few, in segments of at least 1024 positions.  Else 4 waves: up to two workgroups
    // a CU, as many segments as make the six a CU that run in two rounds, of at least 256 positions; beyond, segments of 32
    // tiles, so that the longest sequence is not waited for alone.  All segments have one length (a short sequence has
    // fewer).  us per call in a graph on one state, positions of a segment : us:
    //   BF16  1 x 12 heads of 1000, 26 tokens   8 waves one 7.6, 512: 8.8, 256: 8.0
    //   BF16  1 x 12 of 8000, 16                8 waves 1024: 10.9, 512: 11.4, 2048: 13.7; 4 waves 512: 11.3
    //   FP4   1 x 12 of 1000, 7                 8 waves one 6.2, 256: 7.6; 4 waves one 6.8
    //   FP8   3 x 25 of 1999, 7                 4 waves 256: 9.2, 512: 10.1, one 13.2; 8 waves one 10.9
    //   BF16  8 x 12 ragged of up to 2048, 16   4 waves 256: 9.2, 512: 10.1, one 13.8; 8 waves 11
    //   INT8  8 x 12 ragged of up to 4096, 64   4 waves 1024: 20.5, 512: 22.5, 2048: 24.0, one 28.1; 8 waves one 19.3
    //   INT4 24 x 12 ragged of up to 4096, 32   4 waves 2048: 26.0, 1024: 25.3, one 28.9; 8 waves one 23.0
    //   BF16 16 x 12 ragged of up to 8192, 64   4 waves 1024: 46.6, 512: 50.1, 2048: 50.6, one 53.3
    //   FP8  64 x 12 ragged of up to 1024, 16   4 waves one 16.4, 512: 23.4; 8 waves one 21.0
    //   INT4 64 x 12 ragged of up to 2048, 64   4 waves one 39.4, 1024: 61; 8 waves one 44.6
    // Behind other work (256 MB written before every call), by segments of 512, 1024, 2048, one: BF16 16 x 12 71.8, 72.8,
    // 79.0, 88.6; INT4 24 x 12 34.9, 33.3, 31.8, 35.6; INT8 8 x 12 25.5, 23.8, 26.3, 30.4.
    const int waves = heads <= kFewHeads ? 8 : 4;
    const int tiles = (c.maxT + kSeg - 1) / kSeg;
    int S = 1, seg_tiles = 1;
    if (c.S > 0) {
        if (c.S > kMaxSegments) return KVATTN_ERR_SPLIT;
        S = c.S;
    } else if (c.S < 0) {
        if (-(long long)c.S % kSeg != 0) return KVATTN_ERR_SPLIT;
        seg_tiles = -c.S / kSeg;
        S = (tiles + seg_tiles - 1) / seg_tiles;
        if (S > kMaxSegments) return KVATTN_ERR_SPLIT;
    } else {
        const int tile = c.kv_dtype == KVATTN_KV_F32 ? Kv<KVATTN_KV_F32>::kPos : c.kv_dtype == KVATTN_KV_BF16 ? Kv<KVATTN_KV_BF16>::kPos : 64;
        const int least = waves == 8 ? 16 : heads <= 2 * kCUs ? 4 : 32 * tile / kSeg;
        const long long want = heads <= 2 * kCUs ? 6 * kCUs / heads : kMaxSegments;
        S = (int)std::max<long long>(1, std::min<long long>({want, (tiles + least - 1) / least, 16, kMostWaves / waves / heads}));
        seg_tiles = (tiles + S - 1) / S;
    }
    if (c.B > 65535 || heads * S * waves > kMostWaves) return KVATTN_ERR_SHAPE;
    TreeArgs a{};
    if (S > 1) {
        if (!c.ws) return KVATTN_ERR_WORKSPACE;
        if ((uintptr_t)c.ws & 15u) return KVATTN_ERR_MISALIGNED;
        const auto lay = kvattn_layout::ws_layout((long long)c.num_tokens * c.NH, S, c.ws_bytes);
        if (c.ws_bytes == 0 || lay.bytes > c.ws_bytes) return KVATTN_ERR_WORKSPACE;
        uint8_t* const w = (uint8_t*)c.ws;
        a.counters = (unsigned*)(w + lay.counters);
        a.part_max = (float*)(w + lay.part_max);
        a.part_lse = (float*)(w + lay.part_lse);
        a.part_out = (float*)(w + lay.part_out);
    }
    a.kv = (const uint8_t*)c.kv;
    a.sc = c.scale;
    a.qkv = (const uint8_t*)c.qkv;
    a.out = (uint8_t*)c.out;
    a.table = c.table;
    a.start = c.start;
    a.lens = c.lens;
    a.masks = c.masks;
    a.v_rows = (size_t)c.NH * c.page_rows;
    a.R = c.page_rows;
    a.max_pages = c.max_pages;
    a.num_pages = c.num_pages;
    a.NH = c.NH;
    a.maxT = c.maxT;
    a.words = c.mask_words;
    a.S = S;
    a.seg_tiles = seg_tiles;
    a.num_tokens = c.num_tokens;
    const void* fn = nullptr;
    switch (c.kv_dtype) {
        case KVATTN_KV_F32: fn = kernel_for<KVATTN_KV_F32>(waves); break;
        case KVATTN_KV_BF16: fn = kernel_for<KVATTN_KV_BF16>(waves); break;
        case KVATTN_KV_INT8: fn = kernel_for<KVATTN_KV_INT8>(waves); break;
        case KVATTN_KV_FP8_E4M3: fn = kernel_for<KVATTN_KV_FP8_E4M3>(waves); break;
        case KVATTN_KV_INT4: fn = kernel_for<KVATTN_KV_INT4>(waves); break;
        default: fn = kernel_for<KVATTN_KV_FP4_E2M1>(waves); break;
    }
    void* params[] = {&a};
    return hip_status(hipLaunchKernel(fn, dim3(c.NH * passes, c.B, S), dim3(waves * kWave), params, 0, (hipStream_t)c.stream));
}

}  // namespace kvattn_internal

extern "C" int kvattn_tree_masks(unsigned long long* masks, int* positions, const int* parents, const int* token_start,
                                 const int* lens, int B, int num_tokens, int mask_words, void* stream) {
    if (B < 1 || B > (1 << 20) || num_tokens < 0 || num_tokens > (1 << 30) || mask_words < 1 || mask_words > kMaxMaskWords) return KVATTN_ERR_SHAPE;
    if (num_tokens == 0) return KVATTN_OK;
    if (!masks || !parents || !token_start || (positions && !lens)) return KVATTN_ERR_NULL_POINTER;
    if (((uintptr_t)masks & 7u) || ((uintptr_t)positions & 3u) || ((uintptr_t)parents & 3u) || ((uintptr_t)token_start & 3u) ||
        ((uintptr_t)lens & 3u))
        return KVATTN_ERR_MISALIGNED;
    MaskArgs a{masks, positions, parents, token_start, lens, B, num_tokens, mask_words};
    void* params[] = {&a};
    return hip_status(hipLaunchKernel((const void*)&tree_masks_kernel, dim3((unsigned)B), dim3(kMaxTree), params, 0, (hipStream_t)stream));
}
