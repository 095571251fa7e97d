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

#include <utility>

#include "device_common.h"
#include "token_map.h"

namespace pd {

constexpr int kTokenNative = 0;  // K/V format codes: as q, or the FP8 dtype

template <typename T>
struct TokenMath;

template <>
struct TokenMath<_Float16> {
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
    static constexpr uint32_t kExponents = 0x7C007C00u, kLast = 0x04000400u;  // and their last bits
    static constexpr uint32_t kOnes = 0x3C003C00u;                                     // 1.0 twice
};

template <>
struct TokenMath<__bf16> {
    static constexpr float kOffset = 0.0f, kSlack = 8.0f;
    static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
    }
    template <int KVF>
    static __device__ __forceinline__ u32x2 widen(uint32_t w) {
        bf16x2 a, b;
        if constexpr (KVF == PD_DTYPE_FP8_E4M3) {
            a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
            b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
        } else {
            a = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, false);
            b = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, true);
        }
        return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    }
    static constexpr uint32_t kExponents = 0x7F807F80u, kLast = 0x00800080u;  // and their last bits
    static constexpr uint32_t kOnes = 0x3F803F80u;                                     // 1.0 twice
};

template <>
struct TokenMath<float> {
    static constexpr float kOffset = 0.0f, kSlack = 8.0f;
};

// Whether a 16-byte chunk of QT values, or of FP8 ones as stored (KVF), holds an
// infinity or a NaN: an exponent (E4M3: all bits but the sign) of ones, which one more carries into the sign's place.
template <typename QT, int KVF>
__device__ __forceinline__ bool holds_nonfinite(const u32x4& w) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (KVF == PD_DTYPE_FP8_E4M3) bad |= (((w[i] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
        else if constexpr (KVF == PD_DTYPE_FP8_E5M2) bad |= (((w[i] & 0x7C7C7C7Cu) + 0x04040404u) & 0x80808080u) != 0;
        else if constexpr (sizeof(QT) == 4) bad |= (w[i] & 0x7F800000u) == 0x7F800000u;
        else bad |= (((w[i] & TokenMath<QT>::kExponents) + TokenMath<QT>::kLast) & 0x80008000u) != 0;
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

// Address of an LDS array within the workgroup's LDS.
__device__ __forceinline__ uint32_t lds_address(const char* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)p));
}

template <typename T>
__device__ __forceinline__ T lds_read(uint32_t at) {
    return *(const __attribute__((address_space(3))) T*)at;
}

// Eight bytes of LDS per lane, transposed among each 16 lanes: these address
// four rows of 16 16-bit elements (lane i: row i / 4, elements 4 (i % 4) on), and
// lane i gets element i of each row.
__device__ __forceinline__ u32x2 transposed_read(uint32_t at) {
    typedef __attribute__((address_space(3))) s16x4 LdsVec;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsVec*)at));
}

// The same of bytes: each 16 lanes address eight rows of 16 bytes (lane i: row
// i / 2, bytes 8 (i % 2) on), and lane i gets byte i of each row.
__device__ __forceinline__ u32x2 transposed_bytes(uint32_t at) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i32x2 LdsVec;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((LdsVec*)at));
}

// What a workgroup of the kernel works on.
struct TokenWork {
    int b, kv_head, item;
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
template <typename QT, int KVF, int D>
__device__ __forceinline__ void token_rows_one_by_one(const TokenParams& p, const TokenWork& w, int rows, int first, int step,
                                                      int lane) {
    constexpr int PER = D / kWave;
    constexpr int ES = KVF == kTokenNative ? sizeof(QT) : 1;
    const int32_t* pages = p.table + static_cast<int64_t>(w.b) * p.table_width;
    const char* k_head = static_cast<const char*>(p.k) + static_cast<size_t>(w.kv_head) * D * ES;
    const char* v_head = static_cast<const char*>(p.v) + static_cast<size_t>(w.kv_head) * D * ES;
    for (int i = first; i < rows; i += step) {
        const int row = w.row0 + i;
        if (row >= w.rows) {
            if (p.split == kTokenWhole) store_row_zeros<QT, D>(p, w, row, lane);
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
        if (p.split == kTokenWhole) {
            const float inv = l == 0.0f ? 0.0f : p.v_scale / l;
#pragma unroll
            for (int e = 0; e < PER; ++e)
                static_cast<QT*>(p.out)[at + lane * PER + e] = static_cast<QT>(l == 0.0f ? 0.0f : o[e] * inv);
        } else {
            const int64_t state = token_state(p, w.item, w.kv_head, row);
#pragma unroll
            for (int e = 0; e < PER; ++e) p.numerator[state * D + lane * PER + e] = o[e] * p.v_scale;
            if (lane == 0) *reinterpret_cast<float2*>(p.stats + state * 2) = make_float2(m, l);
        }
    }
}

// ---------------------------------------------------------------------------
// Page ids of a tile of KT tokens from t on: lane i holds that of tokens
// t + 16 i .. + 15. Requested a tile ahead of the rows' own requests, which wait for it.
template <int KT>
__device__ __forceinline__ int tile_pages(const TokenParams& p, const int32_t* pages, int t, int lane) {
    return pages[imin((t + 16 * imin(lane, KT / 16 - 1)) >> p.page_shift, p.table_width - 1)];
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const char* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, bytes, 0x00027000);
}

// 16 bytes per lane from a buffer into LDS at to + kOffset + 16 lane, past the
// registers. In assembly since the compiler, where it knows of such a load, waits for it
// before the next read of any LDS; here wait_for_loads and a barrier come
// before the tile's first read. Nothing is returned in registers.
// kOnce: past the caches, for what is read once.
template <int kOffset, bool kOnce>
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t bytes, uint32_t to, uint32_t offset) {
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    const u32x4 buffer = {static_cast<uint32_t>(at), static_cast<uint32_t>(at >> 32) & 0xFFFFu, bytes, 0x00027000u};
    if constexpr (kOnce)
        asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen nt lds"
                     :
                     : "s"(to), "i"(kOffset), "v"(offset), "s"(buffer)
                     : "memory", "scc");
    else
        asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
                     :
                     : "s"(to), "i"(kOffset), "v"(offset), "s"(buffer)
                     : "memory", "scc");
}

// All loads of this wave but the last kNewer have arrived, those into LDS too.
template <int kNewer = 0>
__device__ __forceinline__ void wait_for_loads() {
    static_assert(kNewer < 64, "the counter's range");
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kNewer) : "memory");
}

// This wave's reads of LDS are done: what they read may be overwritten.
__device__ __forceinline__ void wait_for_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The cache rows of 16 tokens from t on (one page): where they start, and the
// bytes of those before `end` (0 on an invalid page): what lies behind reads as zeros.
struct RowBlock {
    int64_t offset;
    uint32_t bytes;
};

__device__ __forceinline__ RowBlock row_block(const TokenParams& p, int page, int t, int end) {
    const bool valid = static_cast<uint32_t>(page) < static_cast<uint32_t>(p.physical_pages) && t < end;
    const int64_t row = (static_cast<int64_t>(valid ? page : 0) << p.page_shift) + (t & ((1 << p.page_shift) - 1) & ~15);
    return {row * p.kv_row_bytes, valid ? static_cast<uint32_t>(imin(end - t, 16)) * p.kv_row_bytes : 0u};
}

// A tile of KT cache tokens of K or V on its way into LDS, by WAVES waves. It
// goes there directly, as stored, or (kWiden, FP8) through registers, where it is
// widened when it lands.
template <typename QT, int KVF, int D, int WAVES, int KT, bool kWiden, bool kOnce>
struct TileLoad {
    static constexpr bool kFp8 = KVF != kTokenNative;
    static constexpr int SB = D * (kFp8 ? 1 : static_cast<int>(sizeof(QT)));            // bytes of a row in the cache
    static constexpr int RB = kWiden ? D * static_cast<int>(sizeof(QT)) : SB;           // and in LDS
    static constexpr int RPI = 1024 / SB;                        // rows per request of a wave
    static constexpr int NL = KT * SB / 1024 / WAVES;            // requests per wave
    static constexpr int RPW = RPI * NL;                         // neighbouring rows, of 16 or of part of 16 if they are few
    static constexpr int LPR = SB / 16;                          // lanes per row
    static_assert(NL * WAVES * 1024 == KT * SB && 16 % RPI == 0, "whole requests, within 16 tokens");
    static_assert(16 % RPW == 0 || RPW % 16 == 0, "whole blocks of 16 tokens, or parts of one");
    static_assert(!kWiden || kFp8, "what is widened");
    u32x4 raw[kWiden ? NL : 1];

    // ids: the tile's page ids, from lane first_id on; head: the cache from its KV head on; to: the tile's address in LDS.
    __device__ __forceinline__ void request(const TokenParams& p, int ids, int first_id, const char* head, uint32_t to, int t0,
                                            int end, int wave, int lane) {
        request_part(std::make_integer_sequence<int, NL>{}, p, ids, first_id, head, to + wave * (RPW * RB), t0, end, wave, lane);
    }

    template <int... kParts>
    __device__ __forceinline__ void request_part(std::integer_sequence<int, kParts...>, const TokenParams& p, int ids, int first_id,
                                                 const char* head, uint32_t to, int t0, int end, int wave, int lane) {
        (request_one<kParts>(p, ids, first_id, head, to, t0, end, wave, lane), ...);
    }

    template <int kPart>
    __device__ __forceinline__ void request_one(const TokenParams& p, int ids, int first_id, const char* head, uint32_t to, int t0,
                                                int end, int wave, int lane) {
        const int block = wave * RPW / 16 + kPart * RPI / 16;
        const RowBlock rows = row_block(p, __builtin_amdgcn_readlane(ids, first_id + block), t0 + 16 * block, end);
        const int r = wave * RPW % 16 + kPart * RPI % 16 + lane / LPR;
        if constexpr (kWiden) {
            const uint32_t offset = r * p.kv_row_bytes + (lane % LPR) * 16;
            raw[kPart] = __builtin_amdgcn_raw_buffer_load_b128(row_buffer(head + rows.offset, rows.bytes), offset, 0, 0);
        } else {
            // LDS slot `lane` of the request holds the chunk that token_chunk puts there.
            const uint32_t offset = r * p.kv_row_bytes + token_slot_chunk<RB, kFp8>(16 * block + r, lane % LPR) * 16;
            load_to_lds<kPart * RPI * RB, kOnce>(head + rows.offset, rows.bytes, to, offset);
        }
    }

    __device__ __forceinline__ void land(char* tile, int wave, int lane) {
        if constexpr (kWiden) {
#pragma unroll
            for (int jj = 0; jj < NL; ++jj) {
                const int r = RPW * wave + RPI * jj + lane / LPR;
                const u32x4 w = raw[jj];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const u32x2 a = TokenMath<QT>::template widen<KVF>(w[2 * half]);
                    const u32x2 b = TokenMath<QT>::template widen<KVF>(w[2 * half + 1]);
                    *reinterpret_cast<u32x4*>(tile + token_chunk<RB>(r, 2 * (lane % LPR) + half) * 16) = u32x4{a[0], a[1], b[0], b[1]};
                }
            }
        }
    }
};

// Blocks of 16 tokens of a tile on invalid pages, a bit each.
template <int KT>
__device__ __forceinline__ uint32_t invalid_blocks(const TokenParams& p, int ids, int t0, int end, int lane) {
    const bool bad = static_cast<uint32_t>(ids) >= static_cast<uint32_t>(p.physical_pages) && t0 + 16 * lane < end;
    return static_cast<uint32_t>(__ballot(bad)) & ((1u << (KT / 16)) - 1);
}

// A wave's R blocks of 16 rows: q as the first product's operand, what the rows
// see, and their softmax state. KVF: FP8 format of the tiles in LDS, if they are that.
template <typename QT, int KVF, int D, int R>
struct TokenRowsState {
    static constexpr bool kF32 = sizeof(QT) == 4;
    static constexpr bool kFp8 = KVF != kTokenNative;
    static constexpr int RB = D * (kFp8 ? 1 : static_cast<int>(sizeof(QT)));
    static constexpr int KS = D * static_cast<int>(sizeof(QT)) / 64;  // steps of four chunks of the first product
    static constexpr int ND = D / 16;   // blocks of 16 dims of the second
    using Math = TokenMath<QT>;
    u32x4 q[R][KS];
    f32x4 o[R][ND];
    f32x4 l[R];              // sums of weights: all four the whole one (FP32: of the lane's tokens 4 i + e)
    float m[R], most[R];     // scores count from m on, and raise it where they lie above most
    int sees[R];

    __device__ __forceinline__ void open(const TokenParams& p, const TokenWork& w, int first_row, int lane) {
        constexpr int CE = 16 / static_cast<int>(sizeof(QT));
        const int col = lane % 16, quad = lane / 16;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = first_row + r * 16 + col;
            const int token = row / p.group;
            sees[r] = row < w.rows ? imin(w.end, token_sees(p.causal, w.context, w.count, token)) : 0;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                q[r][s] = u32x4{0, 0, 0, 0};
                if (row < w.rows)
                    q[r][s] = *reinterpret_cast<const u32x4*>(static_cast<const QT*>(p.q) +
                                                              token_q_row(p, w.b, w.kv_head, token, row - token * p.group) * D +
                                                              (4 * s + quad) * CE);
            }
            m[r] = 0.0f;
            most[r] = -INFINITY;  // the first token seen sets m
            l[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int d = 0; d < ND; ++d) o[r][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    // q is in its registers: no later read of it waits, and with it for whatever has been requested since.
    __device__ __forceinline__ void arrive() {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[r][s]));
    }

    // Where the lane reads in a tile at `tile` in LDS: bases that constants are added to from one block of tokens to the next.
    // FP8 as stored: rows 16 behind lie in other chunks.
    __device__ __forceinline__ uint32_t k_base(uint32_t tile, int ks, int odd, int lane) const {
        const int col = lane % 16, quad = lane / 16;
        if constexpr (kFp8) return tile + (token_chunk<RB, true>(16 * odd + col, 2 * ks + quad / 2) - odd * RB) * 16 + (quad % 2) * 8;
        else return tile + token_chunk<RB>(col, 4 * ks + quad) * 16;
    }

    // Dim 16 d + col of tokens 4 quad .. + 3 and of those 16 behind, by transposing reads: the 16 lanes of a quad address four
    // rows of four 8-byte pieces (FP8: all eight rows).
    __device__ __forceinline__ uint32_t v_base(uint32_t tile, int d, int lane) const {
        const int col = lane % 16, quad = lane / 16;
        if constexpr (kFp8) return tile + token_chunk<RB, true>(4 * quad + (col / 2) % 4 + (col / 8) * 16, d) * 16 + (col % 2) * 8;
        else return tile + token_chunk<RB>(4 * quad + col / 4, 2 * d + (col % 4) / 2) * 16 + (col % 2) * 8;
    }

    // Scores of a tile of 16 NI tokens, transposed: lane (col, quad) holds row col, tokens 16 i + 4 quad + e.
    template <int NI>
    __device__ __forceinline__ void score(uint32_t k_tile, f32x4 (&s)[R][NI], int lane) {
        uint32_t base[kFp8 ? 2 : 1][KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int odd = 0; odd < (kFp8 ? 2 : 1); ++odd) base[odd][ks] = k_base(k_tile, ks, odd, lane);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                u32x4 kf;
                if constexpr (kFp8) {
                    const u32x2 w = lds_read<u32x2>(base[i % 2][ks] + i * 16 * RB);
                    const u32x2 a = Math::template widen<KVF>(w[0]), b = Math::template widen<KVF>(w[1]);
                    kf = u32x4{a[0], a[1], b[0], b[1]};
                } else {
                    kf = lds_read<u32x4>(base[0][ks] + i * 16 * RB);
                }
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
    }

    // Their weights, and the running maximum. t0: the tile's first token; masked (uniform): some row does not see some token of
    // it. The largest exponent is looked for after the scaling, whose results the maximum takes as they are.
    template <int NI>
    __device__ __forceinline__ void weigh(f32x4 (&s)[R][NI], int t0, bool masked, uint32_t invalid, float scale_log2, int lane) {
        const int quad = lane / 16;
        float top[R];  // of the lane's own
        bool grow = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[r][i][e] = fmaf(s[r][i][e], scale_log2, -m[r]);
            if (masked) {
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool seen = t0 + 16 * i + 4 * quad + e < sees[r] && !(invalid >> i & 1u);
                        s[r][i][e] = seen ? s[r][i][e] : -INFINITY;
                    }
            }
            top[r] = -INFINITY;
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) top[r] = fmaxf(top[r], s[r][i][e]);
            grow |= top[r] > most[r];
        }
        if (__any(grow)) {  // only then do a row's four lanes compare
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float row_top = max_over_lane_groups(top[r]);
                const bool above = row_top > most[r];
                const float up = above ? row_top - Math::kOffset : 0.0f;
                const float alpha = fast_exp2(fminf(-up, 0.0f));  // the first time up may be below 0, with sums of 0 as yet
                most[r] = above ? Math::kSlack : most[r];
                m[r] += up;
                l[r] *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d) o[r][d] *= alpha;
#pragma unroll
                for (int i = 0; i < NI; ++i) s[r][i] -= up;
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < NI; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[r][i][e] = fast_exp2(s[r][i][e]);
                if constexpr (kF32) l[r] += s[r][i];
            }
    }

    // o^T += V^T w^T and l += 1^T w^T, 32 tokens a step (FP32: four, and l on the vector units).
    template <int NI>
    __device__ __forceinline__ void add(uint32_t v_tile, const f32x4 (&s)[R][NI], int lane) {
        if constexpr (kF32) {
            const int col = lane % 16, quad = lane / 16;
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int h = 0; h < ND / 4; ++h) {  // four dims a lane: those of a piece()
                        const f32x4 vf = lds_read<f32x4>(v_tile + token_chunk<RB>(4 * quad + e, 16 * h + col) * 16 + i * 16 * RB);
#pragma unroll
                        for (int d = 0; d < 4; ++d)
#pragma unroll
                            for (int r = 0; r < R; ++r)
                                o[r][4 * h + d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[d], s[r][i][e], o[r][4 * h + d], 0, 0, 0);
                    }
        } else {
            constexpr u32x4 ones = {Math::kOnes, Math::kOnes, Math::kOnes, Math::kOnes};
            uint32_t base[ND];
#pragma unroll
            for (int d = 0; d < ND; ++d) base[d] = v_base(v_tile, d, lane);
#pragma unroll
            for (int u = 0; u < NI / 2; ++u) {
                u32x4 wt[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const f32x4 a = s[r][2 * u], b = s[r][2 * u + 1];
                    wt[r] = u32x4{Math::pack(a[0], a[1]), Math::pack(a[2], a[3]), Math::pack(b[0], b[1]), Math::pack(b[2], b[3])};
                    l[r] = Math::mma(ones, wt[r], l[r]);
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    u32x4 vf;
                    if constexpr (kFp8) {
                        const u32x2 w = transposed_bytes(base[d] + u * 32 * RB);
                        const u32x2 a = Math::template widen<KVF>(w[0]), b = Math::template widen<KVF>(w[1]);
                        vf = u32x4{a[0], a[1], b[0], b[1]};
                    } else {
                        const u32x2 v0 = transposed_read(base[d] + u * 32 * RB);
                        const u32x2 v1 = transposed_read(base[d] + u * 32 * RB + 16 * RB);
                        vf = u32x4{v0[0], v0[1], v1[0], v1[1]};
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r) o[r][d] = Math::mma(vf, wt[r], o[r][d]);
                }
            }
        }
    }

    // Four neighbouring dims of o, and which: piece 0 .. ND - 1 of the lane's row. FP32 V is read four dims at once, so that a
    // block's dims there are every fourth one.
    __device__ __forceinline__ f32x4 piece(int r, int i) const {
        if constexpr (kF32) {
            const int h = i / 4 * 4, e = i % 4;
            return f32x4{o[r][h][e], o[r][h + 1][e], o[r][h + 2][e], o[r][h + 3][e]};
        } else {
            return o[r][i];
        }
    }
    static __device__ __forceinline__ int piece_dim(int i, int lane) {
        return kF32 ? i / 4 * 64 + lane / 16 * 16 + i % 4 * 4 : 16 * i + lane / 16 * 4;
    }

    // The state in LDS, and the other group's of the same rows joined to this one's.
    __device__ __forceinline__ void put(f32x4* to) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int d = 0; d < ND; ++d) to[(r * (ND + 2) + d) * kWave] = o[r][d];
            to[(r * (ND + 2) + ND) * kWave] = l[r];
            to[(r * (ND + 2) + ND + 1) * kWave] = f32x4{m[r], most[r], 0.0f, 0.0f};
        }
    }
    __device__ __forceinline__ void join(const f32x4* from) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const f32x4 head = from[(r * (ND + 2) + ND + 1) * kWave];
            const bool here = most[r] > -INFINITY, there = head[1] > -INFINITY;  // whether they saw any token
            const float top = fmaxf(here ? m[r] : kNoToken, there ? head[0] : kNoToken);
            const float a = here ? fast_exp2(m[r] - top) : 0.0f, b = there ? fast_exp2(head[0] - top) : 0.0f;
            m[r] = top;
            l[r] = l[r] * a + from[(r * (ND + 2) + ND) * kWave] * b;
#pragma unroll
            for (int d = 0; d < ND; ++d) o[r][d] = o[r][d] * a + from[(r * (ND + 2) + d) * kWave] * b;
        }
    }

    // A row's sum of weights, in all of its lanes.
    __device__ __forceinline__ float sum(int r) const {
        if constexpr (kF32) return sum_over_lane_groups((l[r][0] + l[r][1]) + (l[r][2] + l[r][3]));
        else return l[r][0];
    }
};

// The kernel's arguments, read again: what only the end of a kernel needs would
// otherwise be held in scalar registers through its loop, which are too few.
__device__ __forceinline__ TokenParams reloaded_params() {
    const __attribute__((address_space(4))) TokenParams* p =
        (const __attribute__((address_space(4))) TokenParams*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const TokenParams*)p;
}

// Where an item's splits lie: its sequence and the tokens of a split.
struct TokenItem {
    int b, first;  // the sequence, and its first item
    int span;
};

// Sums of x over lanes 0 .. lane: within each row of 16 lanes, then the last lanes' of the rows before.
__device__ __forceinline__ int wave_prefix(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);   // row_shr 1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15: into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast 31: into rows 2 and 3
    return x;
}

// The list of splits, a sequence a lane: splits that end at or before this lane's
// sequence, and the span with which all of them fit p.items.
__device__ __forceinline__ int token_list(const TokenParams& p, int lane, int& span) {
    const int context = lane < p.batch ? token_context(p, lane) : 0;
    for (span = p.split_tokens;; span *= 2) {  // ends: with one split each there are no more than sequences
        const int upto = wave_prefix(token_ceil(context, span));
        if (__builtin_amdgcn_readlane(upto, kWave - 1) <= p.items) return upto;
    }
}

// The sequence of `item` (b = batch if the list is shorter).
__device__ __forceinline__ TokenItem token_item(const TokenParams& p, int item, int lane) {
    TokenItem t;
    if (p.split == kTokenList) {
        const int upto = token_list(p, lane, t.span);
        t.b = imin(__popcll(__ballot(lane < p.batch && upto <= item)), p.batch);
        t.first = t.b > 0 ? __builtin_amdgcn_readlane(upto, t.b - 1) : 0;
    } else {
        const int splits = p.items / p.batch;
        t.b = item / splits;
        t.first = t.b * splits;
        t.span = p.split == kTokenWhole ? p.split_tokens : token_grid_span(splits, p.split_tokens, token_context(p, t.b));
    }
    return t;
}

// The work of a workgroup whose tile has M rows from row0 on; false if no row of it
// sees a token of its split.
template <int M>
__device__ __forceinline__ bool open_work(const TokenParams& p, const TokenCoords& at, TokenWork& w, int& last, int lane) {
    TokenItem t = token_item(p, imin(at.item, p.items - 1), lane);
    if (at.item >= p.items) t.b = p.batch;
    w.b = imin(t.b, p.batch - 1);
    w.item = at.item;
    w.kv_head = at.kv_head;
    w.row0 = at.tile * M;
    w.count = token_count(p, w.b);
    w.context = token_context(p, w.b);
    w.rows = w.count * p.group;
    last = imin(w.row0 + M, w.rows) - 1;
    w.begin = (at.item - t.first) * t.span;
    w.end = last < w.row0 ? 0 : imin(w.begin + t.span, token_sees(p.causal, w.context, w.count, last / p.group));
    return t.b < p.batch && w.begin < w.end;
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of WAVES waves, R blocks of 16 rows each, over tiles of
// KT cache tokens that the waves share through LDS, two of them so that the
// next is on its way while one is used.
// Two GROUPS of such waves take every other tile each, into LDS of their own, and
// join their states at the end. That serves where there is no more than one workgroup of 64
// rows per CU, but too many for splits (us with two groups, with one: FP16, D 64, 8 x
// 96 tokens on 1500 22.6, 25.6; D 128, 300 on 600 14.9, 16.6; FP32, 2 x 200 on 1000
// 80, 87; but 64 on 300, which splits serve, 11.0, 10.3).
// kProductsFirst: waves at their products come before those at their weights, so that
// the two waves of a SIMD fall out of step and one's products run beside the other's
// weights. That takes many equal steps (us with it, without: BF16, D 128, 2048 tokens
// on 8192 227, 239; 1024 on 16384 260, 288; but whole prompts of 2048, whose
// workgroups end at different times, 58.5, 54.7).
// What bounds it: at D 128 the matrix cores (54% busy on 2048 tokens at 8192, 92% of
// a large product's rate in all) and the vector units that they share the SIMDs with.
template <typename QT, int KVF, int D, int R, int WAVES, int KT, int GROUPS, bool kProductsFirst>
__global__ void __launch_bounds__(kWave * WAVES * GROUPS, 2) token_kernel(const TokenParams p) {
    using Rows = TokenRowsState<QT, kTokenNative, D, R>;
    using Load = TileLoad<QT, KVF, D, WAVES, KT, KVF != kTokenNative, false>;
    constexpr int RB = Rows::RB;
    constexpr int M = WAVES * R * 16;
    constexpr int TILE = KT * RB;
    __shared__ __attribute__((aligned(1024))) char tiles[GROUPS * 4 * TILE];  // of each group two of K, two of V

    const int lane = threadIdx.x % kWave;
    const int any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int group = any_wave / WAVES, wave = any_wave % WAVES;
    TokenWork w;
    int last;
    if (!open_work<M>(p, token_coords(p, blockIdx.x), w, last, lane)) {
        if (p.split == kTokenWhole)  // states of such splits are never read
            for (int i = any_wave; i < M; i += WAVES * GROUPS) store_row_zeros<QT, D>(p, w, w.row0 + i, lane);
        return;
    }
    // Cache tokens that every live row of the tile sees.
    const int common = imin(w.end, token_sees(p.causal, w.context, w.count, w.row0 / p.group));
    const bool partial = last - w.row0 != M - 1;
    const char* k_head = static_cast<const char*>(p.k) + static_cast<size_t>(w.kv_head) * Load::SB;
    const char* v_head = static_cast<const char*>(p.v) + static_cast<size_t>(w.kv_head) * Load::SB;
    const int32_t* pages = p.table + static_cast<int64_t>(w.b) * p.table_width;
    Load k_load, v_load;
    constexpr int STEP = GROUPS * KT;
    const int first = w.begin + group * KT;
    int ids = tile_pages<KT>(p, pages, first, lane);
    uint32_t invalid = invalid_blocks<KT>(p, ids, first, w.end, lane);
    char* own = tiles + group * 4 * TILE;
    const uint32_t k_at = lds_address(tiles) + group * 4 * TILE, v_at = k_at + 2 * TILE;
    k_load.request(p, ids, 0, k_head, k_at, first, w.end, wave, lane);
    v_load.request(p, ids, 0, v_head, v_at, first, w.end, wave, lane);
    ids = tile_pages<KT>(p, pages, first + STEP, lane);
    Rows rows;
    rows.open(p, w, w.row0 + wave * R * 16, lane);

    int buffer = 0;
    bool one_by_one = false;
    for (int t = w.begin; t < w.end; t += STEP, buffer ^= 1) {
        const int t0 = t + group * KT;
        char* k_tile = own + buffer * TILE;
        char* v_tile = own + (2 + buffer) * TILE;
        k_load.land(k_tile, wave, lane);
        v_load.land(v_tile, wave, lane);
        wait_for_loads();  // this wave's part of the tile is in LDS
        __syncthreads();   // everyone's part is, and the other tile is no longer read
        const uint32_t here = invalid;
        // Behind the end the request has no rows: it writes zeros that nothing reads.
        invalid = invalid_blocks<KT>(p, ids, t0 + STEP, w.end, lane);
        k_load.request(p, ids, 0, k_head, k_at + (buffer ^ 1) * TILE, t0 + STEP, w.end, wave, lane);
        v_load.request(p, ids, 0, v_head, v_at + (buffer ^ 1) * TILE, t0 + STEP, w.end, wave, lane);
        ids = tile_pages<KT>(p, pages, t0 + 2 * STEP, lane);
        if (t + STEP > common) {  // uniform
            bool bad = false;
            for (int i = wave * kWave + lane; i < TILE / 16; i += WAVES * kWave)
                bad |= holds_nonfinite<QT, kTokenNative>(*reinterpret_cast<const u32x4*>(v_tile + i * 16));
            bad = __builtin_amdgcn_readfirstlane(__syncthreads_or(bad));  // known to be uniform: the loop's state stays in place
            if (bad) {
                one_by_one = true;
                break;
            }
        }
        f32x4 s[R][KT / 16];
        if constexpr (kProductsFirst) __builtin_amdgcn_s_setprio(1);
        rows.score(k_at + buffer * TILE, s, lane);
        if constexpr (kProductsFirst) __builtin_amdgcn_s_setprio(0);
        rows.weigh(s, t0, t0 + KT > common || here != 0 || partial, here, p.scale_log2, lane);
        if constexpr (kProductsFirst) __builtin_amdgcn_s_setprio(1);
        rows.add(v_at + buffer * TILE, s, lane);
        if constexpr (kProductsFirst) __builtin_amdgcn_s_setprio(0);
    }
    wait_for_loads();  // the last request's: nothing may write LDS behind the workgroup's end
    if (one_by_one) {
        token_rows_one_by_one<QT, KVF, D>(p, w, M, any_wave, WAVES * GROUPS, lane);
        return;
    }
    if constexpr (GROUPS == 2) {
        static_assert(WAVES * R * (Rows::ND + 2) * 1024 <= sizeof(tiles), "a group's state in place of the tiles");
        __syncthreads();  // no tile is read any more
        f32x4* state = reinterpret_cast<f32x4*>(tiles) + wave * R * (Rows::ND + 2) * kWave + lane;
        if (group == 1) rows.put(state);
        __syncthreads();
        if (group == 1) return;
        rows.join(state);
    }

    const int col = lane % 16, quad = lane / 16;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float sum = rows.sum(r);
        const int row = w.row0 + (wave * R + r) * 16 + col;
        const int token = row / p.group;
        if (p.split == kTokenWhole) {
            if (token >= p.tokens) continue;
            const float inv = sum == 0.0f ? 0.0f : p.v_scale / sum;
            QT* out = static_cast<QT*>(p.out) + token_q_row(p, w.b, w.kv_head, token, row - token * p.group) * D;
#pragma unroll
            for (int d = 0; d < Rows::ND; ++d) {
                f32x4 x = rows.piece(r, d);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = sum == 0.0f ? 0.0f : x[e] * inv;
                if constexpr (Rows::kF32) *reinterpret_cast<f32x4*>(out + rows.piece_dim(d, lane)) = x;
                else
                    *reinterpret_cast<u32x2*>(out + rows.piece_dim(d, lane)) =
                        u32x2{Rows::Math::pack(x[0], x[1]), Rows::Math::pack(x[2], x[3])};
            }
        } else if (row < w.rows) {
            const int64_t state = token_state(p, w.item, w.kv_head, row);
#pragma unroll
            for (int d = 0; d < Rows::ND; ++d)
                *reinterpret_cast<f32x4*>(p.numerator + state * D + rows.piece_dim(d, lane)) = rows.piece(r, d) * p.v_scale;
            if (quad == 0) *reinterpret_cast<float2*>(p.stats + state * 2) = make_float2(rows.m[r], sum);
        }
    }
}

// ---------------------------------------------------------------------------
// Few rows: every wave streams cache tokens of its own, tiles of 32 or 64 from
// its part of LDS, for all R blocks of 16 rows, and the workgroup's waves of
// one KV head combine at the end. The next K is requested once a tile is scored,
// the next V once it is added, so that a wave always has loads in flight, and nothing
// else in the loop waits for loads: q and the page ids of many tiles are there before
// (us with ids loaded in each step, and so: E4M3, 64 x 4 tokens of up to 4096 76.6, 72.6;
// FP32, 8 x 2 at 2048 34.1, 31.6).
// kOnce: no page is read by two sequences, and K and V stream past the caches (us with,
// without: FP16, 64 sequences of 2048 87.7, 98.9, 32 of up to 4096 67.6, 76.5, 4 of 4096
// 22.8, 23.7; E4M3, 16 of up to 8192 46.4, 49.5).
// What bounds it: memory where a wave has many steps (64 sequences of 2048: 6.4 TB/s);
// with a few, the chain of lengths, page ids and first tiles, and the merge.
template <typename QT, int KVF, int D, int R, int WAVES>
struct StreamShape {
    static constexpr int SB = D * (KVF == kTokenNative ? static_cast<int>(sizeof(QT)) : 1);
    // A wave's tile of K and V is 8 to 32 KB. Rings of two tiles half as long were slower (E4M3, 16 x 8 tokens of up
    // to 8192 47.3 us, so 45.4; 64 x 4 of up to 4096 77.9, 72.6; BF16 the same): every tile has its scalar work.
    static constexpr int KT = SB >= 256 ? 32 : 64;
    static constexpr int TILE = KT * SB;
    static constexpr int SD = D + 4;  // floats from one row's sums to the next: rows begin in other banks
    static constexpr int STATE = R * 16 * SD * 4;
    static constexpr int REGION = 2 * TILE > STATE ? 2 * TILE : STATE;
};

// Page ids of a wave's next tiles of NB blocks of 16 tokens, a block a lane: tiles of every `step`
// tokens from t on. Here, and not where they are used, the wave waits for them, and with them for all that it requested.
template <int NB>
struct PageIds {
    int ids;
    uint64_t invalid;  // blocks on invalid pages

    __device__ __forceinline__ void load(const TokenParams& p, const int32_t* pages, int t, int step, int end, int lane) {
        const int token = t + lane / NB * step + 16 * (lane % NB);
        ids = pages[imin(token >> p.page_shift, p.table_width - 1)];
        asm volatile("" : "+v"(ids));
        invalid = __ballot(static_cast<uint32_t>(ids) >= static_cast<uint32_t>(p.physical_pages) && token < end);
    }

    __device__ __forceinline__ uint32_t invalid_of(int tile) const {
        return static_cast<uint32_t>(invalid >> (tile * NB)) & ((1u << NB) - 1);
    }
};

template <typename QT, int KVF, int D, int R, int WAVES, bool kOnce>
__global__ void __launch_bounds__(kWave * WAVES) token_stream_kernel(const TokenParams p) {
    using Rows = TokenRowsState<QT, KVF, D, R>;
    using Shape = StreamShape<QT, KVF, D, R, WAVES>;
    constexpr int KT = Shape::KT, TILE = Shape::TILE;
    constexpr int NB = KT / 16, TILES = kWave / NB;  // blocks of a tile; tiles whose page ids a wave holds
    using Load = TileLoad<QT, KVF, D, 1, KT, false, kOnce>;
    constexpr int M = R * 16;
    __shared__ __attribute__((aligned(1024))) char regions[WAVES * Shape::REGION];
    __shared__ float2 states[WAVES][M];

    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const TokenCoords at = token_stream_coords(p, blockIdx.x, wave);
    const int slice = wave / p.head_waves, slices = WAVES / p.head_waves;
    TokenWork w;
    int last;
    if (!open_work<M>(p, at, w, last, lane)) {  // the same for all waves
        if (p.split == kTokenWhole && at.item < p.items)  // not the empty ones behind the last item, which have no rows
            for (int i = slice; i < M; i += slices) store_row_zeros<QT, D>(p, w, w.row0 + i, lane);
        return;
    }
    const int common = imin(w.end, token_sees(p.causal, w.context, w.count, w.row0 / p.group));
    const bool partial = last - w.row0 != M - 1;
    const char* k_head = static_cast<const char*>(p.k) + static_cast<size_t>(w.kv_head) * Load::SB;
    const char* v_head = static_cast<const char*>(p.v) + static_cast<size_t>(w.kv_head) * Load::SB;
    const int32_t* pages = p.table + static_cast<int64_t>(w.b) * p.table_width;
    char* region = regions + wave * Shape::REGION;  // K's tile, and V's
    const uint32_t k_at = lds_address(regions) + wave * Shape::REGION, v_at = k_at + TILE;
    const int step = slices * KT;
    const int first = w.begin + slice * KT;

    Load load;
    Rows rows;
    rows.open(p, w, w.row0, lane);
    PageIds<NB> pages_of;
    pages_of.load(p, pages, first, step, w.end, lane);
    rows.arrive();
    load.request(p, pages_of.ids, 0, k_head, k_at, first, w.end, 0, lane);
    load.request(p, pages_of.ids, 0, v_head, v_at, first, w.end, 0, lane);
    uint32_t invalid = pages_of.invalid_of(0);
    int slot = 0;
    bool bad = false;
    for (int t0 = first; t0 < w.end; t0 += step) {
        const bool masked = t0 + KT > common || invalid != 0 || partial;
        f32x4 s[R][KT / 16];
        // Requests behind the end have no rows: they write zeros that nothing reads, and keep the counts the same.
        wait_for_loads<Load::NL>();  // all but V's
        rows.score(k_at, s, lane);
        wait_for_reads();
        slot = (slot + 1) % TILES;
        if (slot == 0) pages_of.load(p, pages, t0 + step, step, w.end, lane);
        load.request(p, pages_of.ids, slot * NB, k_head, k_at, t0 + step, w.end, 0, lane);
        rows.weigh(s, t0, masked, invalid, p.scale_log2, lane);
        wait_for_loads<Load::NL>();  // all but the next K's
        if (t0 + KT > common) {
            for (int i = lane; i < TILE / 16; i += kWave)
                bad |= holds_nonfinite<QT, KVF>(*reinterpret_cast<const u32x4*>(region + TILE + i * 16));
            if (__any(bad)) break;
        }
        rows.add(v_at, s, lane);
        wait_for_reads();
        load.request(p, pages_of.ids, slot * NB, v_head, v_at, t0 + step, w.end, 0, lane);
        invalid = pages_of.invalid_of(slot);
    }
    wait_for_loads();
    const TokenParams late = reloaded_params();
    if (__syncthreads_or(bad)) {
        token_rows_one_by_one<QT, KVF, D>(late, w, M, slice, slices, lane);
        return;
    }

    // The waves' states, into their own parts of LDS.
    float* sums = reinterpret_cast<float*>(region);
    const int col = lane % 16, quad = lane / 16;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float sum = rows.sum(r);
#pragma unroll
        for (int d = 0; d < Rows::ND; ++d)
            *reinterpret_cast<f32x4*>(sums + (r * 16 + col) * Shape::SD + rows.piece_dim(d, lane)) = rows.piece(r, d);
        if (quad == 0) states[wave][r * 16 + col] = make_float2(rows.m[r], sum);
    }
    __syncthreads();
    // Four dims of a row a lane; all waves of the head together, and a few states' reads at once.
    constexpr int LPR = D / 4, RPW = kWave / LPR;  // lanes per row, rows per wave
    constexpr int kAtOnce = WAVES / 2;             // divides the slices of either number of heads per workgroup
    const int dim = (lane % LPR) * 4;
    const int mate = wave % late.head_waves;       // the first wave of the same head
    for (int i = slice * RPW + lane / LPR; i < M; i += slices * RPW) {
        const int row = w.row0 + i, token = row / late.group;
        if (token >= late.tokens) continue;
        float m = kNoToken, l = 0.0f;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int j0 = 0; j0 < slices; j0 += kAtOnce)
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const float2 st = states[mate + (j0 + j) * late.head_waves][i];
                m = fmaxf(m, st.y != 0.0f ? st.x : kNoToken);
            }
        for (int j0 = 0; j0 < slices; j0 += kAtOnce) {
            f32x4 x[kAtOnce];
            float a[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const int from = mate + (j0 + j) * late.head_waves;
                const float2 st = states[from][i];
                a[j] = st.y != 0.0f ? fast_exp2(st.x - m) : 0.0f;
                l = fmaf(st.y, a[j], l);
                x[j] = *reinterpret_cast<const f32x4*>(regions + from * Shape::REGION + (i * Shape::SD + dim) * 4);
            }
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(x[j][e], a[j], o[e]);
        }
        if (late.split == kTokenWhole) {
            QT* out = static_cast<QT*>(late.out) + token_q_row(late, w.b, w.kv_head, token, row - token * late.group) * D + dim;
            const float inv = l == 0.0f ? 0.0f : late.v_scale / l;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = l == 0.0f ? 0.0f : o[e] * inv;
            if constexpr (Rows::kF32) *reinterpret_cast<f32x4*>(out) = o;
            else
                *reinterpret_cast<u32x2*>(out) = u32x2{Rows::Math::pack(o[0], o[1]), Rows::Math::pack(o[2], o[3])};
        } else if (row < w.rows) {
            const int64_t state = token_state(late, w.item, w.kv_head, row);
            *reinterpret_cast<f32x4*>(late.numerator + state * D + dim) = o * late.v_scale;
            if (dim == 0) *reinterpret_cast<float2*>(late.stats + state * 2) = make_float2(m, l);
        }
    }
}

// ---------------------------------------------------------------------------
// Splits of each row into its output: kWaves waves per row (1 or 4), which take
// parts of its splits. Four dims a lane, so that kWave / (D / 4) states are read
// at once, kUnroll times over and together with the statistics: a row's reads, of
// lengths, then of states, are what the kernel waits for.
template <typename QT, int D, int kWaves>
__global__ void __launch_bounds__(256) token_merge_kernel(const TokenParams p) {
    constexpr int LPS = D / 4;          // lanes per state
    constexpr int SPW = kWave / LPS;    // states per read
    constexpr int kUnroll = 16 / SPW;   // reads of 16 states
    __shared__ f32x4 sums[kWaves][LPS];
    __shared__ float2 parts[kWaves];
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (4 / kWaves) + wave / kWaves;
    const int64_t rows = static_cast<int64_t>(p.batch) * p.tokens * p.query_heads;
    if (item >= rows) return;  // with several waves per row, all of a workgroup or none
    const uint32_t bt = static_cast<uint32_t>(item / p.query_heads);
    const int head = static_cast<int>(item - static_cast<int64_t>(bt) * p.query_heads);
    const int b = static_cast<int>(bt / p.tokens), token = static_cast<int>(bt - static_cast<uint32_t>(b) * p.tokens);
    const int kv_head = head / p.group;
    int first, span;  // the sequence's splits
    if (p.split == kTokenList) {
        const int upto = token_list(p, lane, span);
        first = b > 0 ? __builtin_amdgcn_readlane(upto, b - 1) : 0;
    } else {
        const int splits = p.items / p.batch;
        first = b * splits;
        span = token_grid_span(splits, p.split_tokens, token_context(p, b));
    }
    const int count = token_count(p, b), context = token_context(p, b);
    const int sees = token < count ? token_sees(p.causal, context, count, token) : 0;
    const int all = token_ceil(sees, span);  // splits that hold a token it sees
    const int64_t next = token_state(p, 1, 0, 0);  // from one split's state to the next one's
    const int share = token_ceil(all, kWaves), from0 = (wave % kWaves) * share;
    const int live = imin(all - from0, share);     // this wave's, from from0 on
    const int64_t state = token_state(p, first, kv_head, token * p.group + head - kv_head * p.group) + from0 * next;
    const float2* stats = reinterpret_cast<const float2*>(p.stats) + state;
    const float* numerator = p.numerator + state * D + (lane % LPS) * 4;

    float m = kNoToken, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < live; s0 += kWave) {
        const int here = imin(live - s0, kWave);
        f32x4 x[kUnroll];
        auto read = [&](int s) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int at = s0 + imin(s + u * SPW + lane / LPS, here - 1);
                x[u] = *reinterpret_cast<const f32x4*>(numerator + at * next * D);
            }
        };
        const float2 st = stats[(s0 + imin(lane, here - 1)) * next];
        read(0);
        const bool filled = lane < here && st.y != 0.0f;
        const float top = fmaxf(m, wave_max(filled ? st.x : kNoToken));
        const float alpha = fast_exp2(m - top);  // of the 64 splits before
        m = top;
        const float a = filled ? fast_exp2(st.x - m) : 0.0f;
        l = fmaf(l, alpha, filled ? st.y * a : 0.0f);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = alpha != 0.0f ? o[e] * alpha : 0.0f;
        for (int s = 0; s < here; s += SPW * kUnroll) {
            if (s > 0) read(s);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int from = s + u * SPW + lane / LPS;
                const float weight = __shfl(a, from & (kWave - 1));
                // A state of weight 0 (none at all, or one with nothing in it) adds nothing, whatever it holds.
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = from < here && weight != 0.0f ? fmaf(x[u][e], weight, o[e]) : o[e];
            }
        }
    }
    l = wave_sum(l);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (LPS == 16) o[e] += __shfl_xor(o[e], 16);
        o[e] += __shfl_xor(o[e], 32);
    }
    if constexpr (kWaves > 1) {
        if (lane < LPS) sums[wave][lane] = o;
        if (lane == 0) parts[wave] = make_float2(m, l);
        __syncthreads();
        if (wave > 0) return;
        float top = kNoToken;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) top = fmaxf(top, parts[i].y != 0.0f ? parts[i].x : kNoToken);
        l = 0.0f;
        o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            const float a = parts[i].y != 0.0f ? fast_exp2(parts[i].x - top) : 0.0f;
            l = fmaf(parts[i].y, a, l);
            const f32x4 x = sums[i][lane % LPS];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = a != 0.0f ? fmaf(x[e], a, o[e]) : o[e];
        }
    }
    if (lane < LPS) {
        QT* out = static_cast<QT*>(p.out) + item * D + lane * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = l == 0.0f ? 0.0f : o[e] / l;
        if constexpr (sizeof(QT) == 4) *reinterpret_cast<f32x4*>(out) = o;
        else
            *reinterpret_cast<u32x2*>(out) = u32x2{TokenMath<QT>::pack(o[0], o[1]), TokenMath<QT>::pack(o[2], o[3])};
    }
}

}  // namespace pd

#endif  // PAGED_DECODE_TOKEN_KERNELS_H
