// Attention of several tokens per sequence over the paged cache, as templates:
// each tokens_*.hip translation unit instantiates those of one q format and
// head dimension.
//
// For the rows of a tile (query tokens x heads of one KV head) and cache
// tokens t, in one pass over the cache tokens with a running maximum:
//   s = K q (scaled, in log2 units), hidden tokens at -infinity
//   m' = max(m, max s), w = 2^(s - m'), l = l 2^(m - m') + sum w, o = o 2^(m - m') + w V
// and out = o / l. Both products run on the matrix cores transposed, K q^T and
// V^T w^T, so that a lane's four scores per 16 tokens are one row's: sums over
// tokens stay in the lane but for its three partners, the weights are the
// second product's operand as they stand, and rescaling o needs no exchange.
#ifndef PAGED_DECODE_TOKEN_KERNELS_H
#define PAGED_DECODE_TOKEN_KERNELS_H

#include "device_common.h"
#include "token_map.h"

namespace pd {

constexpr int kTokenNative = 0;  // K/V format codes: as q, or the FP8 dtype

template <typename T>
struct TokenMath;

template <>
struct TokenMath<_Float16> {
    typedef f16x8 Frag;
    // Weights lie below 2^14 and the running maximum's own at 2^6, so that those 2^-20 of it keep 11 bits.
    static constexpr float kOffset = 6.0f, kSlack = 14.0f;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
    }
    template <int KVF>
    static __device__ __forceinline__ u32x2 widen(uint32_t w) {  // four FP8 values, exact
        f16x2 a, b;
        if constexpr (KVF == PD_DTYPE_FP8_E4M3) {
            a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
            b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
        } else {
            a = __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, false);
            b = __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, true);
        }
        return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    }
    static constexpr uint32_t kExponents = 0x7C007C00u, kExponent = 0x7C00u;
};

template <>
struct TokenMath<__bf16> {
    typedef bf16x8 Frag;
    static constexpr float kOffset = 0.0f, kSlack = 8.0f;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
    }
    template <int KVF>
    static __device__ __forceinline__ u32x2 widen(uint32_t w) {  // FP8 values are the top halves of their FP32 form
        f32x2 a, b;
        if constexpr (KVF == PD_DTYPE_FP8_E4M3) {
            a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
            b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        } else {
            a = __builtin_amdgcn_cvt_pk_f32_bf8(w, false);
            b = __builtin_amdgcn_cvt_pk_f32_bf8(w, true);
        }
        const float a0 = a[0], a1 = a[1], b0 = b[0], b1 = b[1];
        return u32x2{(__builtin_bit_cast(uint32_t, a0) >> 16) | (__builtin_bit_cast(uint32_t, a1) & 0xFFFF0000u),
                     (__builtin_bit_cast(uint32_t, b0) >> 16) | (__builtin_bit_cast(uint32_t, b1) & 0xFFFF0000u)};
    }
    static constexpr uint32_t kExponents = 0x7F807F80u, kExponent = 0x7F80u;
};

template <>
struct TokenMath<float> {
    static constexpr float kOffset = 0.0f, kSlack = 8.0f;
};

// Whether a 16-byte chunk holds an infinity or a NaN.
template <typename QT>
__device__ __forceinline__ bool holds_nonfinite(const u32x4& w) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(QT) == 4) {
            bad |= (w[i] & 0x7F800000u) == 0x7F800000u;
        } else {
            constexpr uint32_t kLow = TokenMath<QT>::kExponent, kHigh = kLow << 16;
            bad |= (w[i] & kLow) == kLow || (w[i] & kHigh) == kHigh;
        }
    }
    return bad;
}

// One stored K/V element as FP32.
template <typename QT, int KVF>
__device__ __forceinline__ float stored_value(const char* p, int i) {
    if constexpr (KVF == kTokenNative) return static_cast<float>(reinterpret_cast<const QT*>(p)[i]);
    const int byte = reinterpret_cast<const uint8_t*>(p)[i];
    f32x2 f;
    if constexpr (KVF == PD_DTYPE_FP8_E5M2) f = __builtin_amdgcn_cvt_pk_f32_bf8(byte, false);
    else f = __builtin_amdgcn_cvt_pk_f32_fp8(byte, false);
    return f[0];
}

// Eight bytes of LDS per lane, transposed among each 16 lanes: these address
// four rows of 16 16-bit elements (lane i: row i / 4, elements 4 (i % 4) on), and
// lane i gets element i of each row.
__device__ __forceinline__ u32x2 transposed_read(const char* p) {
    typedef __attribute__((address_space(3))) s16x4 LdsVec;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsVec*)p));
}

// What a workgroup of the kernel works on.
struct TokenWork {
    int b, kv_head, split;
    int row0;       // first row of the tile
    int rows;       // live rows of the sequence (tokens x group)
    int count, context;
    int begin, end; // cache tokens of the split that some row of the tile sees
};

template <typename QT, int D>
__device__ __forceinline__ void store_row_zeros(const TokenParams& p, const TokenWork& w, int row, int lane) {
    const int token = row / p.group;
    if (token >= p.tokens) return;
    QT* out = static_cast<QT*>(p.out) + token_q_row(p, w.b, w.kv_head, token, row - token * p.group) * D;
    for (int i = lane; i < D; i += kWave) out[i] = static_cast<QT>(0.0f);
}

// The rows of a tile one by one, a wave each, on the vector units: for tiles
// in which a token that some rows see and others do not has an infinity or NaN in
// V, since 0 * V would carry it into the rows that do not see it.
template <typename QT, int KVF, int D, int WAVES, int M>
__device__ __forceinline__ void token_rows_one_by_one(const TokenParams& p, const TokenWork& w, int wave, int lane) {
    constexpr int PER = D / kWave;
    constexpr int ES = KVF == kTokenNative ? sizeof(QT) : 1;
    const int32_t* pages = p.table + static_cast<int64_t>(w.b) * p.table_width;
    const char* k_head = static_cast<const char*>(p.k) + static_cast<size_t>(w.kv_head) * D * ES;
    const char* v_head = static_cast<const char*>(p.v) + static_cast<size_t>(w.kv_head) * D * ES;
    for (int i = wave; i < M; i += WAVES) {
        const int row = w.row0 + i;
        if (row >= w.rows) {
            if (p.splits == 1) store_row_zeros<QT, D>(p, w, row, lane);
            continue;
        }
        const int token = row / p.group;
        const int64_t at = token_q_row(p, w.b, w.kv_head, token, row - token * p.group) * D;
        const int limit = imin(w.end, token_sees(p.causal, w.context, w.count, token));
        float q[PER], o[PER], m = kNoToken, l = 0.0f;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            q[e] = static_cast<float>(static_cast<const QT*>(p.q)[at + lane * PER + e]);
            o[e] = 0.0f;
        }
        for (int t = w.begin; t < limit; ++t) {
            const int page = pages[t >> p.page_shift];
            if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.physical_pages)) continue;
            const int64_t offset = ((static_cast<int64_t>(page) << p.page_shift) + (t & ((1 << p.page_shift) - 1))) * p.kv_row_bytes;
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < PER; ++e) s = fmaf(stored_value<QT, KVF>(k_head + offset, lane * PER + e), q[e], s);
            s = wave_sum(s) * p.scale_log2;
            const float top = fmaxf(m, s);
            const float alpha = fast_exp2(m - top), weight = fast_exp2(s - top);
            m = top;
            l = l * alpha + weight;
#pragma unroll
            for (int e = 0; e < PER; ++e) o[e] = o[e] * alpha + weight * stored_value<QT, KVF>(v_head + offset, lane * PER + e);
        }
        if (p.splits == 1) {
            const float inv = l == 0.0f ? 0.0f : p.v_scale / l;
#pragma unroll
            for (int e = 0; e < PER; ++e)
                static_cast<QT*>(p.out)[at + lane * PER + e] = static_cast<QT>(l == 0.0f ? 0.0f : o[e] * inv);
        } else {
            const int64_t state = token_state(p, w.b, w.kv_head, row, w.split);
#pragma unroll
            for (int e = 0; e < PER; ++e) p.numerator[state * D + lane * PER + e] = o[e] * p.v_scale;
            if (lane == 0) *reinterpret_cast<float2*>(p.stats + state * 2) = make_float2(m, l);
        }
    }
}

// A workgroup of WAVES waves, R blocks of 16 rows each, over tiles of KT cache
// tokens that the waves share through LDS.
template <typename QT, int KVF, int D, int R, int WAVES, int KT>
__global__ void __launch_bounds__(kWave * WAVES) token_kernel(const TokenParams p) {
    constexpr bool kF32 = sizeof(QT) == 4;
    constexpr int ES = KVF == kTokenNative ? static_cast<int>(sizeof(QT)) : 1;  // stored element
    constexpr int RB = D * static_cast<int>(sizeof(QT));  // bytes of a tile row in LDS
    constexpr int CPR = RB / 16;
    constexpr int NI = KT / 16;         // blocks of 16 cache tokens
    constexpr int KS = RB / 64;         // steps of four chunks of the first product
    constexpr int ND = D / 16;          // blocks of 16 dims of the second
    constexpr int M = WAVES * R * 16;
    constexpr int CE = 16 / static_cast<int>(sizeof(QT));  // elements of a chunk
    using Math = TokenMath<QT>;
    __shared__ __attribute__((aligned(16))) char k_tile[KT * RB];
    __shared__ __attribute__((aligned(16))) char v_tile[KT * RB];

    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane % 16, quad = lane / 16;

    TokenWork w;
    const TokenCoords at = token_coords(p, blockIdx.x);
    w.b = at.b;
    w.kv_head = at.kv_head;
    w.split = at.split;
    w.row0 = at.tile * M;
    w.count = token_count(p, w.b);
    w.context = token_context(p, w.b);
    w.rows = w.count * p.group;
    const int last = imin(w.row0 + M, w.rows) - 1;
    const int span = token_split(p.splits, p.split_tokens, w.context);
    w.begin = w.split * span;
    w.end = last < w.row0 ? 0 : imin(w.begin + span, token_sees(p.causal, w.context, w.count, last / p.group));
    if (w.begin >= w.end) {  // nothing to see; states of such splits are never read
        if (p.splits == 1)
            for (int i = wave; i < M; i += WAVES) store_row_zeros<QT, D>(p, w, w.row0 + i, lane);
        return;
    }
    // Cache tokens that every live row of the tile sees.
    const int common = token_sees(p.causal, w.context, w.count, w.row0 / p.group);

    const int32_t* pages = p.table + static_cast<int64_t>(w.b) * p.table_width;
    const char* k_head = static_cast<const char*>(p.k) + static_cast<size_t>(w.kv_head) * D * ES;
    const char* v_head = static_cast<const char*>(p.v) + static_cast<size_t>(w.kv_head) * D * ES;

    // This lane's rows: q as the first product's operand, and what they see.
    u32x4 q[R][KS];
    int sees[R];
    int64_t out_at[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = w.row0 + (wave * R + r) * 16 + col;
        const int token = row / p.group;
        sees[r] = row < w.rows ? imin(w.end, token_sees(p.causal, w.context, w.count, token)) : 0;
        out_at[r] = token < p.tokens ? token_q_row(p, w.b, w.kv_head, token, row - token * p.group) * D : -1;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            q[r][s] = u32x4{0, 0, 0, 0};
            if (row < w.rows)
                q[r][s] = *reinterpret_cast<const u32x4*>(static_cast<const QT*>(p.q) + out_at[r] + (4 * s + quad) * CE);
        }
    }
    f32x4 o[R][ND];
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = kNoToken;
        l[r] = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[r][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    for (int t0 = w.begin; t0 < w.end; t0 += KT) {
        __syncthreads();
        // K and V rows of the tile into LDS; rows behind the end and on invalid pages are zeros.
        for (int i = threadIdx.x; i < KT * CPR; i += WAVES * kWave) {
            const int r = i / CPR, c = i % CPR;
            const int t = t0 + r;
            u32x4 kc = {0, 0, 0, 0}, vc = {0, 0, 0, 0};
            if (t < w.end) {
                const int page = pages[t >> p.page_shift];
                if (static_cast<uint32_t>(page) < static_cast<uint32_t>(p.physical_pages)) {
                    const int64_t row = (static_cast<int64_t>(page) << p.page_shift) + (t & ((1 << p.page_shift) - 1));
                    const int64_t offset = row * p.kv_row_bytes + c * CE * ES;
                    if constexpr (KVF == kTokenNative) {
                        kc = *reinterpret_cast<const u32x4*>(k_head + offset);
                        vc = *reinterpret_cast<const u32x4*>(v_head + offset);
                    } else {
                        const u32x2 kw = *reinterpret_cast<const u32x2*>(k_head + offset);
                        const u32x2 vw = *reinterpret_cast<const u32x2*>(v_head + offset);
                        const u32x2 k0 = Math::template widen<KVF>(kw[0]), k1 = Math::template widen<KVF>(kw[1]);
                        const u32x2 v0 = Math::template widen<KVF>(vw[0]), v1 = Math::template widen<KVF>(vw[1]);
                        kc = u32x4{k0[0], k0[1], k1[0], k1[1]};
                        vc = u32x4{v0[0], v0[1], v1[0], v1[1]};
                    }
                }
            }
            const int at = token_chunk<RB>(r, c) * 16;
            *reinterpret_cast<u32x4*>(k_tile + at) = kc;
            *reinterpret_cast<u32x4*>(v_tile + at) = vc;
        }
        uint32_t invalid = 0;  // blocks of 16 tokens on invalid pages
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int t = t0 + 16 * i;
            if (t < w.end && static_cast<uint32_t>(pages[t >> p.page_shift]) >= static_cast<uint32_t>(p.physical_pages))
                invalid |= 1u << i;
        }
        __syncthreads();
        if (t0 + KT > common) {  // uniform
            bool bad = false;
            for (int i = threadIdx.x; i < KT * CPR; i += WAVES * kWave)
                bad |= holds_nonfinite<QT>(*reinterpret_cast<const u32x4*>(v_tile + i * 16));
            if (__syncthreads_or(bad)) {
                token_rows_one_by_one<QT, KVF, D, WAVES, M>(p, w, wave, lane);
                return;
            }
        }

        // Scores, transposed: lane (col, quad) holds row col, tokens 16 i + 4 quad + e.
        f32x4 s[R][NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(k_tile + token_chunk<RB>(16 * i + col, 4 * ks + quad) * 16);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if constexpr (kF32) {
                        const f32x4 a = __builtin_bit_cast(f32x4, kf), b = __builtin_bit_cast(f32x4, q[r][ks]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[r][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], s[r][i], 0, 0, 0);
                    } else {
                        s[r][i] = Math::mma(kf, q[r][ks], s[r][i]);
                    }
                }
            }
        }
        const bool masked = t0 + KT > imin(common, w.end) || invalid != 0 || last - w.row0 != M - 1;  // uniform
        float top[R];
        bool grow = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (masked) {
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = t0 + 16 * i + 4 * quad + e;
                        const bool seen = t < sees[r] && !(invalid >> i & 1u);
                        s[r][i][e] = seen ? s[r][i][e] : -INFINITY;
                    }
            }
            float x = s[r][0][0];
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) x = fmaxf(x, s[r][i][e]);
            top[r] = max_over_lane_groups(x) * p.scale_log2;
            grow |= top[r] > m[r] + Math::kSlack;
        }
        if (__any(grow)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float next = top[r] > m[r] + Math::kSlack ? top[r] - Math::kOffset : m[r];
                const float alpha = fast_exp2(m[r] - next);
                m[r] = next;
                l[r] *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[r][d] *= alpha;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[r][i][e] = fast_exp2(fmaf(s[r][i][e], p.scale_log2, -m[r]));
                    l[r] += s[r][i][e];
                }

        // o^T += V^T w^T, 32 tokens a step (FP32: four).
        if constexpr (kF32) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const int row = 16 * i + 4 * quad + e;
                        const float vf = *reinterpret_cast<const float*>(
                            v_tile + token_chunk<RB>(row, 4 * d + col / 4) * 16 + (col % 4) * 4);
#pragma unroll
                        for (int r = 0; r < R; ++r)
                            o[r][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf, s[r][i][e], o[r][d], 0, 0, 0);
                    }
        } else {
#pragma unroll
            for (int u = 0; u < NI / 2; ++u) {
                u32x4 wt[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const f32x4 a = s[r][2 * u], b = s[r][2 * u + 1];
                    wt[r] = u32x4{Math::pack(a[0], a[1]), Math::pack(a[2], a[3]), Math::pack(b[0], b[1]), Math::pack(b[2], b[3])};
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    // Lane (col, quad) gets dim 16 d + col of tokens 4 quad .. + 3, by a transposing read: the 16 lanes of a
                    // quad address four rows of four 8-byte pieces.
                    const int row = 32 * u + 4 * quad + col / 4;
                    const int piece = 2 * d + (col % 4) / 2;
                    const u32x2 v0 = transposed_read(v_tile + token_chunk<RB>(row, piece) * 16 + (col % 2) * 8);
                    const u32x2 v1 = transposed_read(v_tile + token_chunk<RB>(row + 16, piece) * 16 + (col % 2) * 8);
                    const u32x4 vf = {v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
                    for (int r = 0; r < R; ++r) o[r][d] = Math::mma(vf, wt[r], o[r][d]);
                }
            }
        }
    }

#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float sum = sum_over_lane_groups(l[r]);
        const int row = w.row0 + (wave * R + r) * 16 + col;
        if (p.splits == 1) {
            if (out_at[r] < 0) continue;
            const float inv = sum == 0.0f ? 0.0f : p.v_scale / sum;
            QT* out = static_cast<QT*>(p.out) + out_at[r];
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                f32x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = sum == 0.0f ? 0.0f : o[r][d][e] * inv;
                if constexpr (kF32) *reinterpret_cast<f32x4*>(out + 16 * d + 4 * quad) = x;
                else *reinterpret_cast<u32x2*>(out + 16 * d + 4 * quad) = u32x2{Math::pack(x[0], x[1]), Math::pack(x[2], x[3])};
            }
        } else if (row < w.rows) {
            const int64_t state = token_state(p, w.b, w.kv_head, row, w.split);
#pragma unroll
            for (int d = 0; d < ND; ++d)
                *reinterpret_cast<f32x4*>(p.numerator + state * D + 16 * d + 4 * quad) = o[r][d] * p.v_scale;
            if (quad == 0) *reinterpret_cast<float2*>(p.stats + state * 2) = make_float2(m[r], sum);
        }
    }
}

// Splits of each row into its output: a wave per row.
template <typename QT, int D>
__global__ void __launch_bounds__(256) token_merge_kernel(const TokenParams p) {
    constexpr int PER = D / kWave;
    const int lane = threadIdx.x % kWave;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    const int64_t rows = static_cast<int64_t>(p.batch) * p.tokens * p.query_heads;
    if (item >= rows) return;
    const int head = static_cast<int>(item % p.query_heads);
    const int64_t bt = item / p.query_heads;
    const int b = static_cast<int>(bt / p.tokens), token = static_cast<int>(bt % p.tokens);
    const int kv_head = head / p.group;
    const int count = token_count(p, b), context = token_context(p, b);
    const int sees = token < count ? token_sees(p.causal, context, count, token) : 0;
    const int span = token_split(p.splits, p.split_tokens, context);
    const int live = (sees + span - 1) / span;  // splits that hold a token it sees
    const int64_t state = token_state(p, b, kv_head, token * p.group + head - kv_head * p.group, 0);
    const float2* stats = reinterpret_cast<const float2*>(p.stats) + state;
    float m = kNoToken;
    for (int s = 0; s < live; ++s) {
        const float2 st = stats[s];
        m = st.y != 0.0f ? fmaxf(m, st.x) : m;
    }
    float l = 0.0f, o[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] = 0.0f;
    for (int s = 0; s < live; ++s) {
        const float2 st = stats[s];
        if (st.y == 0.0f) continue;
        const float a = fast_exp2(st.x - m);
        l += st.y * a;
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] = fmaf(p.numerator[(state + s) * D + lane * PER + e], a, o[e]);
    }
    QT* out = static_cast<QT*>(p.out) + item * D + lane * PER;
#pragma unroll
    for (int e = 0; e < PER; ++e) out[e] = static_cast<QT>(l == 0.0f ? 0.0f : o[e] / l);
}

}  // namespace pd

#endif  // PAGED_DECODE_TOKEN_KERNELS_H
