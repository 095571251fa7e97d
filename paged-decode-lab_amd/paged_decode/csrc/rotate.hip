// Norms of queries and keys for each head with the position rotation in the
// same pass, and the paged KV-cache append that takes keys that way into the
// cache (quantised where the cache holds FP8).
//
// For a head x of D dims at position p:
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w                  (w given)
//   (y_a, y_b) <- s * (y_a cos t - y_b sin t, y_a sin t + y_b cos t),  t = p f_i
// for each pair i of the first R dims; dims from R on are left as they are.
// Everything is FP32 and rounded once, to the output's type; the angle is a
// product in 64 bits, reduced to an eighth of a turn there, since FP32 would
// lose 0.06 rad at position 10^6.
//
// The kernels are bound by memory where there are many tokens and by a launch
// where there are few.
#include "device_common.h"
#include "rotate_map.h"

namespace pd {
namespace {

constexpr int kRotateWaves = 4;         // waves of a workgroup
constexpr int kAdvanceWaves = 8;        // and of one that holds a whole sequence's new tokens
constexpr int kMaxPairs = 64;           // rotated pairs of a head
constexpr double kTurnsPerRadian = 0.15915494309189533576888;

__device__ __forceinline__ void load_eight(const float* p, float (&f)[8]) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[e] = a[e];
        f[4 + e] = b[e];
    }
}

template <typename T>
__device__ __forceinline__ void load_eight(const T* p, float (&f)[8]) {
    typedef T Vec __attribute__((ext_vector_type(8)));
    const Vec v = *reinterpret_cast<const Vec*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(v[e]);
}

// Stores past the caches: with ordinary ones the same kernel took 46 us instead
// of 40 for four prompts of 2048 tokens (168 MB), 38 instead of 34 for the FP8 append of 8 x 1024.
__device__ __forceinline__ void store_eight(float* p, const float (&f)[8]) {
    __builtin_nontemporal_store(f32x4{f[0], f[1], f[2], f[3]}, reinterpret_cast<f32x4*>(p));
    __builtin_nontemporal_store(f32x4{f[4], f[5], f[6], f[7]}, reinterpret_cast<f32x4*>(p) + 1);
}

template <typename T>
__device__ __forceinline__ void store_eight(T* p, const float (&f)[8]) {
    typedef T Vec __attribute__((ext_vector_type(8)));
    Vec v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<T>(f[e]);
    __builtin_nontemporal_store(v, reinterpret_cast<Vec*>(p));
}

// FP8 bytes of x / scale, saturated to the largest finite value (infinities
// too); NaN stays NaN.
template <int FMT>
__device__ __forceinline__ uint32_t four_fp8(float a, float b, float c, float d) {
    int w = 0;
    if constexpr (FMT == PD_DTYPE_FP8_E4M3) {
        w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    } else {
        w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
        w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
    }
    return static_cast<uint32_t>(w);
}

template <int FMT>
__device__ __forceinline__ void store_eight_fp8(char* p, const float (&f)[8], float scale, float largest) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float y = f[e] / scale;
        x[e] = y != y ? y : fminf(fmaxf(y, -largest), largest);
    }
    __builtin_nontemporal_store(u32x2{four_fp8<FMT>(x[0], x[1], x[2], x[3]), four_fp8<FMT>(x[4], x[5], x[6], x[7])},
                                reinterpret_cast<u32x2*>(p));
}

// cos and sin of 2 pi * turns: the nearest quarter turn is taken off in 64
// bits, so that FP32 sees an eighth of a turn at most.
__device__ __forceinline__ float2 turn_cos_sin(double turns) {
    const double quarters = rint(4.0 * turns);
    const float rest = static_cast<float>(2.0 * (turns - 0.25 * quarters));
    float s, c;
    sincospif(rest, &s, &c);
    const int quadrant = static_cast<int>(static_cast<long long>(quarters)) & 3;
    const float cs = quadrant & 1 ? s : c, sn = quadrant & 1 ? c : s;
    return make_float2(quadrant == 1 || quadrant == 2 ? -cs : cs, quadrant >= 2 ? -sn : sn);
}

__device__ __forceinline__ int64_t append_row(const AppendParams& a, const int32_t* pages, int64_t pos) {
    const int64_t entry = append_table_entry(a, pos);
    if (entry < 0) return -1;
    return append_cache_row(a, pages[entry], pos);
}

__device__ __forceinline__ int live_tokens(const RotateParams& p, int b) {
    return p.counts == nullptr ? p.tokens : imin(imax(p.counts[b], 0), p.tokens);
}

// Whether `count` tokens from position `base` on all map to valid cache rows.
// Every lane of the wave calls it; a lane looks at every 64th page.
__device__ __forceinline__ bool sequence_fits(const AppendParams& a, const int32_t* pages, int64_t base, int count, int lane) {
    if (count == 0) return true;
    if (base < 0 || base + count > a.capacity) return false;
    const int64_t last = (base + count - 1) >> a.page_shift;
    bool fits = true;
    for (int64_t e = (base >> a.page_shift) + lane; e <= last; e += kWave)
        fits &= static_cast<uint32_t>(pages[e]) < static_cast<uint32_t>(a.physical_pages);
    return __all(fits);
}

// One wave's head group `group` of token `token` of sequence b at position pos;
// turns: the wave's (cos, sin) pairs in LDS. The heads are requested before the
// angles are worked out, which they cover: left out, those save 0 to 3%.
template <typename T, int CF, int D>
__device__ __forceinline__ void rotate_token(const RotateParams& p, int b, int token, int64_t pos, bool live, int64_t cache_row,
                                             int group, int lane, float2* turns) {
    constexpr int LPH = D / kRotateLaneDims;  // lanes per head
    const int j = lane % LPH;
    const ChunkPair ch = rotate_chunks(p.rotary_dim, p.interleaved, j);
    const bool turned = j < p.rotary_dim / kRotateLaneDims;
    const int head = group * (kWave / LPH) + lane / LPH;
    const bool is_q = head < p.q_heads;
    const bool is_k = !is_q && head < p.q_heads + p.kv_heads;
    const int h = is_q ? head : is_k ? head - p.q_heads : head - p.q_heads - p.kv_heads;
    const int64_t out_token = static_cast<int64_t>(b) * p.tokens + token;
    float x[8], y[8];
    if (head < p.heads && live) {
        const TokenRows& rows = is_q ? p.q : is_k ? p.k : p.v;
        const T* in = reinterpret_cast<const T*>(rows.data) + token_row_offset(rows, b, token, h, D);
        load_eight(in + ch.first, x);
        load_eight(in + ch.second, y);
    }
    float cs[8], sn[8];
    if (p.rotary_dim > 0) {
        if (lane < p.rotary_dim / 2) {
            const float2 t = turn_cos_sin(static_cast<double>(pos) * (p.frequencies[lane] * kTurnsPerRadian));
            turns[lane] = make_float2(t.x * p.turn_scale, t.y * p.turn_scale);
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (turned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float2 t = turns[8 * j + e];
            cs[e] = t.x;
            sn[e] = t.y;
        }
    }
    if (head >= p.heads) return;
    if (!live) {  // rows behind a sequence's tokens: zeros in q, the cache as it was
        if (is_q) {
            T* out = reinterpret_cast<T*>(p.q_out) + (out_token * p.q_heads + h) * D;
            const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            store_eight(out + ch.first, zero);
            store_eight(out + ch.second, zero);
        }
        return;
    }
    const void* weight = is_q ? p.q_weight : is_k ? p.k_weight : nullptr;
    if (weight != nullptr) {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], fmaf(y[e], y[e], sum));
        sum += dpp_move<kDppQuadSwap1>(sum);
        sum += dpp_move<kDppQuadSwap2>(sum);
        if constexpr (LPH == 8) sum += dpp_move<kDppRowHalfMirror>(sum);
        const float inv = 1.0f / sqrtf(fmaf(sum, p.inv_dim, p.eps));
        const int64_t w0 = static_cast<int64_t>(h) * (is_q ? p.q_weight_stride : p.k_weight_stride);
        float wx[8], wy[8];
        if (p.weight_f32) {
            load_eight(static_cast<const float*>(weight) + w0 + ch.first, wx);
            load_eight(static_cast<const float*>(weight) + w0 + ch.second, wy);
        } else {
            load_eight(static_cast<const T*>(weight) + w0 + ch.first, wx);
            load_eight(static_cast<const T*>(weight) + w0 + ch.second, wy);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = x[e] * inv * wx[e];
            y[e] = y[e] * inv * wy[e];
        }
    }
    if (turned && (is_q || is_k)) {
        if (p.interleaved) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float a = x[2 * e], c = x[2 * e + 1], d = y[2 * e], f = y[2 * e + 1];
                x[2 * e] = a * cs[e] - c * sn[e];
                x[2 * e + 1] = a * sn[e] + c * cs[e];
                y[2 * e] = d * cs[4 + e] - f * sn[4 + e];
                y[2 * e + 1] = d * sn[4 + e] + f * cs[4 + e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float a = x[e], c = y[e];
                x[e] = a * cs[e] - c * sn[e];
                y[e] = a * sn[e] + c * cs[e];
            }
        }
    }
    if (is_q || CF < 0) {
        T* out = reinterpret_cast<T*>(is_q ? p.q_out : p.k_out) + (out_token * (is_q ? p.q_heads : p.kv_heads) + h) * D;
        store_eight(out + ch.first, x);
        store_eight(out + ch.second, y);
    } else if constexpr (CF >= 0) {
        if (cache_row >= 0) {
            constexpr int ES = CF == PD_DTYPE_FP8_E4M3 || CF == PD_DTYPE_FP8_E5M2 ? 1 : static_cast<int>(sizeof(T));
            char* out = (is_k ? p.cache.k_cache : p.cache.v_cache) + cache_row * p.cache.row_bytes +
                        static_cast<int64_t>(h) * D * ES;
            if constexpr (ES == 1) {
                const float scale = is_k ? p.k_scale : p.v_scale;
                store_eight_fp8<CF>(out + ch.first, x, scale, p.largest);
                store_eight_fp8<CF>(out + ch.second, y, scale, p.largest);
            } else {
                store_eight(reinterpret_cast<T*>(out) + ch.first, x);
                store_eight(reinterpret_cast<T*>(out) + ch.second, y);
            }
        }
    }
}

// Cache formats: -1 none (k_out), 0 the tokens' own type, or an FP8 dtype code.
// kAdvance: positions from lengths, all or nothing per sequence (the lengths
// are advanced by a launch behind this one).
template <typename T, int CF, int D, bool kAdvance>
__global__ void __launch_bounds__(kWave * kRotateWaves) rotate_kernel(const RotateParams p) {
    __shared__ float2 turns[kRotateWaves][kMaxPairs];
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t item = blockIdx.x * kRotateWaves + wave;
    const uint32_t tokens = static_cast<uint32_t>(p.batch) * p.tokens;  // at most 2^31 items (host)
    const uint32_t at = item / p.head_groups;
    if (at >= tokens) return;
    const int b = at / p.tokens, token = at % p.tokens;
    const bool live = token < live_tokens(p, b);
    int64_t row = -1, pos;
    if constexpr (kAdvance) pos = static_cast<int64_t>(p.cache.lengths[b]) + token;
    else pos = p.per_token_positions ? p.positions[at] : static_cast<int64_t>(p.positions[b]) + token;
    if constexpr (CF >= 0) {
        const int32_t* pages = p.cache.table + static_cast<int64_t>(b) * p.cache.table_width;
        if (!kAdvance || sequence_fits(p.cache, pages, pos - token, live_tokens(p, b), lane)) row = append_row(p.cache, pages, pos);
    }
    rotate_token<T, CF, D>(p, b, token, pos, live, row, item % p.head_groups, lane, turns[wave]);
}

// A whole sequence's new tokens in one workgroup, which then advances its length.
template <typename T, int CF, int D>
__global__ void __launch_bounds__(kWave * kAdvanceWaves) rotate_advance_kernel(const RotateParams p) {
    __shared__ float2 turns[kAdvanceWaves][kMaxPairs];
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int b = blockIdx.x;
    const int32_t* pages = p.cache.table + static_cast<int64_t>(b) * p.cache.table_width;
    const int64_t base = p.cache.lengths[b];
    const int count = live_tokens(p, b);
    const bool fits = sequence_fits(p.cache, pages, base, count, lane);
    for (int i = wave; i < p.tokens * p.head_groups; i += kAdvanceWaves) {
        const int token = i / p.head_groups;
        const int64_t row = fits && token < count ? append_row(p.cache, pages, base + token) : -1;
        rotate_token<T, CF, D>(p, b, token, base + token, token < count, row, i % p.head_groups, lane, turns[wave]);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();  // every wave has read lengths[b] before it changes
    if (threadIdx.x == 0 && fits) p.cache.lengths[b] = static_cast<int32_t>(base + count);
}

// lengths[b] += counts[b] for the sequences whose tokens fit: the launch behind
// rotate_kernel<.., kAdvance>, which has read the lengths. One wave per sequence.
__global__ void __launch_bounds__(kWave) advance_lengths_kernel(const RotateParams p) {
    const int b = blockIdx.x;
    const int64_t base = p.cache.lengths[b];
    const int count = live_tokens(p, b);
    const bool fits = sequence_fits(p.cache, p.cache.table + static_cast<int64_t>(b) * p.cache.table_width, base, count,
                                    threadIdx.x);
    if (threadIdx.x == 0 && fits) p.cache.lengths[b] = static_cast<int32_t>(base + count);
}

// ---------------------------------------------------------------------------
// Host side.

// Sequences of up to this many head-group passes are appended by one workgroup
// each, which also advances the length; longer ones by as many workgroups as
// they fill, with a launch behind them for the lengths.
constexpr int kAdvanceMaxPasses = 4 * kAdvanceWaves;

size_t type_size(int dtype) { return dtype == PD_DTYPE_F32 ? 4 : 2; }

bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

// 0 if the rows can be read 16 bytes at a time.
int check_rows(const pd_token_rows* r, int dtype, int heads) {
    if (!r->data) return PD_ERR_NULL_POINTER;
    const int64_t unit = 16 / static_cast<int64_t>(type_size(dtype));
    if (misaligned(r->data) || r->batch_stride % unit != 0 || r->token_stride % unit != 0) return PD_ERR_SHAPE;
    if (heads < 1 || heads > 65535) return PD_ERR_SHAPE;
    // Strides may be 0 (one row for several tokens), never negative; offsets stay far inside 63 bits.
    const int64_t limit = int64_t{1} << 40;
    if (r->batch_stride < 0 || r->token_stride < 0 || r->batch_stride > limit || r->token_stride > limit) return PD_ERR_SHAPE;
    return PD_OK;
}

int check_rotation(const pd_rotation* r, int dtype, int head_dim) {
    if (!r) return PD_ERR_NULL_POINTER;
    if (r->rotary_dim < 0 || r->rotary_dim > head_dim || r->rotary_dim % kRotateLaneDims != 0) return PD_ERR_SHAPE;
    if (r->rotary_dim > 0 && !r->frequencies) return PD_ERR_NULL_POINTER;
    if (r->style != PD_ROTATE_HALF && r->style != PD_ROTATE_INTERLEAVED) return PD_ERR_SHAPE;
    if (!(r->scale - r->scale == 0.0f)) return PD_ERR_SHAPE;  // finite
    if (r->q_weight || r->k_weight) {
        if (r->weight_dtype != dtype && r->weight_dtype != PD_DTYPE_F32) return PD_ERR_DTYPE;
        if (!(r->eps >= 0.0f) || !(r->eps - r->eps == 0.0f)) return PD_ERR_SHAPE;
        if (misaligned(r->q_weight) || misaligned(r->k_weight)) return PD_ERR_SHAPE;
    }
    return PD_OK;
}

RotateParams rotate_params(const pd_rotation* r, int batch, int tokens, int head_dim) {
    RotateParams p{};
    p.frequencies = r->frequencies;
    p.q_weight = r->q_weight;
    p.k_weight = r->k_weight;
    p.eps = r->eps;
    p.inv_dim = 1.0f / static_cast<float>(head_dim);
    p.turn_scale = r->scale;
    p.k_scale = p.v_scale = 1.0f;
    p.batch = batch;
    p.tokens = tokens;
    p.rotary_dim = r->rotary_dim;
    p.interleaved = r->style == PD_ROTATE_INTERLEAVED;
    p.weight_f32 = r->weight_dtype == PD_DTYPE_F32;
    p.q_weight_stride = r->q_weight_per_head ? head_dim : 0;
    p.k_weight_stride = r->k_weight_per_head ? head_dim : 0;
    return p;
}

TokenRows token_rows(const pd_token_rows* r) {
    if (r == nullptr) return TokenRows{};
    return TokenRows{static_cast<const char*>(r->data), r->batch_stride, r->token_stride};
}

// A wave takes one head group of one token. Waves of several groups, which would
// work out a token's angles once, were as fast from two groups on and slower with the whole
// token (us, four prompts of 2048 tokens: 37.4, 39.6 with two, 43.3 with all five).
int plan_rotate(RotateParams& p, int head_dim) {
    const int hpw = rotate_heads_per_wave(head_dim);
    p.head_groups = (p.heads + hpw - 1) / hpw;
    // A launch holds 2^32 threads.
    return static_cast<int64_t>(p.batch) * p.tokens * p.head_groups <= (int64_t{1} << 26) - kRotateWaves ? PD_OK : PD_ERR_SHAPE;
}

uint32_t rotate_blocks(const RotateParams& p) {
    const int64_t waves = static_cast<int64_t>(p.batch) * p.tokens * p.head_groups;
    return static_cast<uint32_t>((waves + kRotateWaves - 1) / kRotateWaves);
}

template <typename T, int CF, int D>
int launch_rotate(RotateParams& p, bool advance, hipStream_t stream) {
    int status = plan_rotate(p, D);
    if (status != PD_OK) return status;
    if constexpr (CF >= 0) {
        if (advance && static_cast<int64_t>(p.tokens) * p.head_groups <= kAdvanceMaxPasses) {
            hipLaunchKernelGGL((rotate_advance_kernel<T, CF, D>), dim3(p.batch), dim3(kWave * kAdvanceWaves), 0, stream, p);
            return hipGetLastError() == hipSuccess ? PD_OK : PD_ERR_LAUNCH;
        }
        if (advance) {
            hipLaunchKernelGGL((rotate_kernel<T, CF, D, true>), dim3(rotate_blocks(p)), dim3(kWave * kRotateWaves), 0, stream, p);
            hipLaunchKernelGGL(advance_lengths_kernel, dim3(p.batch), dim3(kWave), 0, stream, p);
            return hipGetLastError() == hipSuccess ? PD_OK : PD_ERR_LAUNCH;
        }
    }
    hipLaunchKernelGGL((rotate_kernel<T, CF, D, false>), dim3(rotate_blocks(p)), dim3(kWave * kRotateWaves), 0, stream, p);
    return hipGetLastError() == hipSuccess ? PD_OK : PD_ERR_LAUNCH;
}

template <int CF>
int dispatch_rotate(RotateParams& p, int dtype, int head_dim, bool advance, hipStream_t stream) {
    if (dtype == PD_DTYPE_F32) {
        if constexpr (CF > 0) return PD_ERR_DTYPE;
        else return head_dim == 64 ? launch_rotate<float, CF, 64>(p, advance, stream)
                                   : launch_rotate<float, CF, 128>(p, advance, stream);
    }
    if (dtype == PD_DTYPE_F16)
        return head_dim == 64 ? launch_rotate<_Float16, CF, 64>(p, advance, stream)
                              : launch_rotate<_Float16, CF, 128>(p, advance, stream);
    return head_dim == 64 ? launch_rotate<__bf16, CF, 64>(p, advance, stream)
                          : launch_rotate<__bf16, CF, 128>(p, advance, stream);
}

bool valid_scale(float s) { return s > 0.0f && s - s == 0.0f; }

// Shared by the two append entries: `advance` takes positions from lengths.
int append_rotated(const pd_rotation* rotation, const pd_token_rows* q, const pd_token_rows* k, const pd_token_rows* v,
                   int dtype, const int32_t* table, const int32_t* positions, int32_t* lengths, const int32_t* counts,
                   void* q_out, void* k_cache, void* v_cache, int cache_dtype, float k_scale, float v_scale, int batch,
                   int tokens, int query_heads, int kv_heads, int head_dim, int page_size, int table_width,
                   int physical_pages, int max_context, void* stream) {
    const bool advance = lengths != nullptr;
    if (!rotation || !k || !v || !table || (!positions && !lengths) || !k_cache || !v_cache) return PD_ERR_NULL_POINTER;
    if (q && !q_out) return PD_ERR_NULL_POINTER;
    if (dtype < PD_DTYPE_F32 || dtype > PD_DTYPE_BF16) return PD_ERR_DTYPE;
    const bool fp8 = cache_dtype == PD_DTYPE_FP8_E4M3 || cache_dtype == PD_DTYPE_FP8_E5M2;
    if (!(cache_dtype == dtype || (fp8 && dtype != PD_DTYPE_F32))) return PD_ERR_DTYPE;
    if (!valid_scale(k_scale) || !valid_scale(v_scale)) return PD_ERR_DTYPE;
    if (!fp8 && (k_scale != 1.0f || v_scale != 1.0f)) return PD_ERR_DTYPE;
    if (batch < 1 || batch > 65535 || tokens < 1 || tokens > 65535 || kv_heads < 1 || kv_heads > 65535) return PD_ERR_SHAPE;
    if (head_dim != 64 && head_dim != 128) return PD_ERR_SHAPE;
    if (page_size != 16 && page_size != 32) return PD_ERR_SHAPE;
    if (table_width < 1 || table_width > 65536 || physical_pages < 1) return PD_ERR_SHAPE;
    if (advance && (max_context < 0 || max_context > (1 << 20))) return PD_ERR_SHAPE;
    if (misaligned(k_cache) || misaligned(v_cache) || misaligned(q_out)) return PD_ERR_SHAPE;
    int status = check_rotation(rotation, dtype, head_dim);
    if (status == PD_OK && q) status = check_rows(q, dtype, query_heads);
    if (status == PD_OK) status = check_rows(k, dtype, kv_heads);
    if (status == PD_OK) status = check_rows(v, dtype, kv_heads);
    if (status != PD_OK) return status;
    RotateParams p = rotate_params(rotation, batch, tokens, head_dim);
    p.q = token_rows(q);
    p.k = token_rows(k);
    p.v = token_rows(v);
    p.q_out = static_cast<char*>(q_out);
    p.positions = positions;
    p.counts = counts;
    p.q_heads = q ? query_heads : 0;
    p.kv_heads = kv_heads;
    p.heads = p.q_heads + 2 * kv_heads;
    p.k_scale = k_scale;
    p.v_scale = v_scale;
    p.largest = cache_dtype == PD_DTYPE_FP8_E4M3 ? 448.0f : 57344.0f;
    AppendParams& a = p.cache;
    a.table = table;
    a.lengths = lengths;
    a.k_cache = static_cast<char*>(k_cache);
    a.v_cache = static_cast<char*>(v_cache);
    a.tokens = tokens;
    a.table_width = table_width;
    a.page_shift = page_size == 16 ? 4 : 5;
    a.physical_pages = physical_pages;
    a.capacity = static_cast<int64_t>(table_width) << a.page_shift;
    if (advance) a.capacity = std::min<int64_t>(a.capacity, max_context);
    a.row_bytes = static_cast<uint32_t>(static_cast<size_t>(kv_heads) * head_dim * (fp8 ? 1 : type_size(dtype)));
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (cache_dtype == PD_DTYPE_FP8_E4M3) return dispatch_rotate<PD_DTYPE_FP8_E4M3>(p, dtype, head_dim, advance, s);
    if (cache_dtype == PD_DTYPE_FP8_E5M2) return dispatch_rotate<PD_DTYPE_FP8_E5M2>(p, dtype, head_dim, advance, s);
    return dispatch_rotate<0>(p, dtype, head_dim, advance, s);
}

}  // namespace
}  // namespace pd

extern "C" {

int pd_rotate_heads(const pd_rotation* rotation, const pd_token_rows* q, const pd_token_rows* k, int dtype,
                    const int32_t* positions, int positions_per_token, void* q_out, void* k_out, int batch, int tokens,
                    int query_heads, int kv_heads, int head_dim, void* stream) {
    using namespace pd;
    if (!rotation || !q || !positions || !q_out || (k && !k_out)) return PD_ERR_NULL_POINTER;
    if (dtype < PD_DTYPE_F32 || dtype > PD_DTYPE_BF16) return PD_ERR_DTYPE;
    if (batch < 1 || batch > 65535 || tokens < 1 || tokens > 65535) return PD_ERR_SHAPE;
    if (head_dim != 64 && head_dim != 128) return PD_ERR_SHAPE;
    if (misaligned(q_out) || misaligned(k_out)) return PD_ERR_SHAPE;
    int status = check_rotation(rotation, dtype, head_dim);
    if (status == PD_OK) status = check_rows(q, dtype, query_heads);
    if (status == PD_OK && k) status = check_rows(k, dtype, kv_heads);
    if (status != PD_OK) return status;
    RotateParams p = rotate_params(rotation, batch, tokens, head_dim);
    p.q = token_rows(q);
    p.k = token_rows(k);
    p.q_out = static_cast<char*>(q_out);
    p.k_out = static_cast<char*>(k_out);
    p.positions = positions;
    p.per_token_positions = positions_per_token != 0;
    p.q_heads = query_heads;
    p.kv_heads = k ? kv_heads : 0;
    p.heads = p.q_heads + p.kv_heads;
    return dispatch_rotate<-1>(p, dtype, head_dim, false, static_cast<hipStream_t>(stream));
}

int pd_append_rotated(const pd_rotation* rotation, const pd_token_rows* q, const pd_token_rows* k,
                      const pd_token_rows* v, int dtype, const int32_t* table, const int32_t* positions,
                      const int32_t* counts, void* q_out, void* k_cache, void* v_cache, int cache_dtype, float k_scale,
                      float v_scale, int batch, int tokens, int query_heads, int kv_heads, int head_dim, int page_size,
                      int table_width, int physical_pages, void* stream) {
    return pd::append_rotated(rotation, q, k, v, dtype, table, positions, nullptr, counts, q_out, k_cache, v_cache,
                              cache_dtype, k_scale, v_scale, batch, tokens, query_heads, kv_heads, head_dim, page_size,
                              table_width, physical_pages, 0, stream);
}

int pd_append_rotated_advance(const pd_rotation* rotation, const pd_token_rows* q, const pd_token_rows* k,
                              const pd_token_rows* v, int dtype, const int32_t* table, int32_t* lengths,
                              const int32_t* counts, void* q_out, void* k_cache, void* v_cache, int cache_dtype,
                              float k_scale, float v_scale, int batch, int tokens, int query_heads, int kv_heads,
                              int head_dim, int page_size, int table_width, int physical_pages, int max_context,
                              void* stream) {
    if (!lengths) return PD_ERR_NULL_POINTER;
    return pd::append_rotated(rotation, q, k, v, dtype, table, nullptr, lengths, counts, q_out, k_cache, v_cache,
                              cache_dtype, k_scale, v_scale, batch, tokens, query_heads, kv_heads, head_dim, page_size,
                              table_width, physical_pages, max_context, stream);
}

}  // extern "C"
