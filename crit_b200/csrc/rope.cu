// The step in front of the cache: each head of the queries and keys divided by its root mean square and weighted, its pairs
// turned by angles of the token's position(s), and (when the call writes) the keys and values encoded into their pages, in
// one launch.
//
//   y = x / sqrt(mean x^2 + eps) * (offset + w)                              where a weight is given, else y = x
//   (a, b) -> magnitude * (a cos - b sin, b cos + a sin)                     pairs (i, rotary / 2 + i), or (2 i, 2 i + 1)
//   angle of pair i = positions[axes[i]][token] * frequencies[i]             (axes NULL: positions[token])
//
// A block takes one token, or a few where a token has few heads.  Its threads first make the tokens' sines and cosines in
// shared memory, once for every head: the angle is a product in FP64 (a position of 2^20 times a frequency loses 2^-4 of a
// radian in FP32), reduced to a part of a turn there and handed to sincospi in FP32.  Then 8, 16 or 32 lanes share a row of up to 64,
// 128 or 256 elements: a lane holds four pairs, two vectors of four elements, so nothing crosses lanes but the sum of
// squares.  A row that goes to a page is laid out again through shared memory, eight neighbouring elements a lane, and
// encoded from its FP32 values as crit_b200_append encodes rows (16-bit pages, E4M3, INT8 and 4-bit codes).
// All sums are FP32; a result is rounded once.  Every element is read and written once: bound by HBM for prompt chunks, by
// the launch for decode steps.
#include <type_traits>

#include "int4.cuh"

namespace crit_b200 {

constexpr int ROPE_WARPS = 8;
constexpr int ROPE_MAX_TOKENS = 16;         // tokens a block takes

template <typename T>
__device__ __forceinline__ void load4(const T* src, float (&x)[4]) {
    if constexpr (sizeof(T) == 4) {
        const float4 v = *reinterpret_cast<const float4*>(src);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(src);
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
            x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
        } else {
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
            x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* dst, const float (&x)[4]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]));
    }
}

__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
    if (dtype == CRIT_B200_DTYPE_BF16) return __bfloat162float(((const __nv_bfloat16*)w)[i]);
    if (dtype == CRIT_B200_DTYPE_FP16) return __half2float(((const __half*)w)[i]);
    return ((const float*)w)[i];
}

// A lane's eight neighbouring elements of a row (lane `part` of the row's lanes, `span` of them) into the row's page slot.
// Every lane of the warp comes here: lanes without elements (or whose row is not written) with live false.
__device__ __forceinline__ void encode_row(const crit_b200_append_params& a, const float (&x)[8], bool live, bool is_v, int64_t slot, int h,
                                           int dim, int part, int span) {
    const int64_t row = slot * a.kv_heads + h;
    char* pages = (char*)(is_v ? a.value_pages : a.key_pages);
    if (a.kind == CRIT_B200_KIND_INT4) {
        uint32_t byte;
        const uint32_t w = int4_quantise(x, byte);
        if (!live) return;
        reinterpret_cast<uint32_t*>(pages)[row * (dim >> 3) + part] = w;
        if ((part & 3) == 0) reinterpret_cast<uint8_t*>(is_v ? a.value_scales : a.key_scales)[row * (dim >> 5) + (part >> 2)] = (uint8_t)byte;
        return;
    }
    if (a.kind == CRIT_B200_KIND_16BIT) {
        if (!live) return;
        if (a.page_dtype == CRIT_B200_DTYPE_FP32) {
            float4* dst = reinterpret_cast<float4*>((float*)pages + row * dim + part * 8);
            dst[0] = make_float4(x[0], x[1], x[2], x[3]), dst[1] = make_float4(x[4], x[5], x[6], x[7]);
            return;
        }
        const bool bf16 = a.page_dtype == CRIT_B200_DTYPE_BF16;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = bf16 ? pack2<true>(x[2 * i], x[2 * i + 1]) : pack2<false>(x[2 * i], x[2 * i + 1]);
        *reinterpret_cast<uint4*>(pages + (row * dim + part * 8) * 2) = make_uint4(w[0], w[1], w[2], w[3]);
        return;
    }
    float div = is_v ? a.value_multiplier : a.key_multiplier;
    if (a.kind != CRIT_B200_KIND_FP8) {                      // a scale a row: its largest magnitude over 448 or 127
        float amax = 0.f;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) nan |= x[i] != x[i], amax = fmaxf(amax, fabsf(x[i]));
        int bits = nan ? 0x7fffffff : __float_as_int(amax);
        for (int o = 1; o < span; o <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
        const float s = __fdiv_rn(__int_as_float(bits), a.kind == CRIT_B200_KIND_FP8_ROW ? 448.f : 127.f);
        div = bits > 0x7f800000 ? __int_as_float(0x7fc00000) : fmaxf(s, 1e-30f);
        if (live && part == 0) (is_v ? a.value_scales : a.key_scales)[row] = div;
    }
    if (!live) return;
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = __fdiv_rn(x[i], div);
        uint32_t c;
        if (a.kind == CRIT_B200_KIND_INT8) c = (uint8_t)(int8_t)fminf(fmaxf(rintf(y), -127.f), 127.f);
        else c = float_to_e4m3(y);
        w[i >> 2] |= c << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(pages + row * dim + part * 8) = make_uint2(w[0], w[1]);
}

// LANES: of a row (8, 16 or 32: the widest head has up to 8 elements a lane).
template <typename T, int LANES, bool WRITE>
__global__ void __launch_bounds__(ROPE_WARPS * 32) norm_rope_kernel(const crit_b200_norm_rope_params p, const crit_b200_append_params a, const int per_block) {
    constexpr int ROWS = 32 / LANES;                         // rows a warp holds at once
    extern __shared__ float rope_smem[];
    float2* turns = reinterpret_cast<float2*>(rope_smem);    // [tokens of the block][rotary / 2] (cos, sin)
    const int half = p.rotary >> 1;
    const int64_t token0 = (int64_t)blockIdx.x * per_block;
    const int tokens = (int)(p.tokens - token0 < per_block ? p.tokens - token0 : per_block);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane % LANES, sub = lane / LANES;
    float* relay = rope_smem + 2 * per_block * half + (warp * ROWS + sub) * (LANES * 8 + 4);

    for (int i = threadIdx.x; i < tokens * half; i += ROPE_WARPS * 32) {
        const int tok = i / half, pair = i - tok * half;
        const int axis = p.axes ? p.axes[pair] : 0;
        float2 turn = make_float2(0.f, 0.f);
        if (axis >= 0 && axis < p.n_axes) {
            const double at = (double)p.positions[(int64_t)axis * p.axis_stride + token0 + tok] * (double)p.frequencies[pair];
            // at / (2 pi) less its whole turns: 1 / (2 pi) as a sum of two FP64 numbers, the product's rounding put back
            const double turns_of = at * 0.15915494309189535;
            const double rest = fma(at, 0.15915494309189535, -turns_of) + at * -9.839338337591243e-18;
            float s, c;
            sincospif((float)(2.0 * ((turns_of - rint(turns_of)) + rest)), &s, &c);
            turn = make_float2(c * p.magnitude, s * p.magnitude);
        } else if (p.status) {
            atomicExch(p.status, CRIT_B200_STATUS_BOUNDS);   // an axis that positions has not: the pair becomes zeros
        }
        turns[i] = turn;
    }
    __syncthreads();

    const int row_heads = p.q_heads + p.kv_heads + (WRITE && a.values ? p.kv_heads : 0);
    const int rows = tokens * row_heads;
    for (int row0 = warp * ROWS; row0 < rows; row0 += ROPE_WARPS * ROWS) {
        const int row = row0 + sub;
        const bool here = row < rows;
        const int tok = here ? row / row_heads : 0;
        const int head = row - tok * row_heads;
        const bool is_q = head < p.q_heads, is_v = head >= p.q_heads + p.kv_heads;
        const int h = is_q ? head : (is_v ? head - p.q_heads - p.kv_heads : head - p.q_heads);
        const int64_t t = token0 + tok;
        const int dim = is_v ? a.value_dim : p.head_dim;
        // the lane's two vectors of four elements: of a turned chunk the pairs' halves (or four neighbouring pairs)
        const bool turned = !is_v && part * 4 < half;
        const int e0 = turned ? (p.interleaved ? part * 8 : part * 4) : (is_v ? part * 8 : p.rotary + (part - (half >> 2)) * 8);
        const int e1 = turned && !p.interleaved ? half + part * 4 : e0 + 4;
        const bool live = here && part * 8 < dim;
        float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
        if (live) {
            const T* src = is_q ? (const T*)p.q + t * p.q_stride_token + (int64_t)h * p.q_stride_head
                                : (is_v ? (const T*)a.values + t * a.value_stride_token + (int64_t)h * a.value_stride_head
                                        : (const T*)p.keys + t * p.key_stride_token + (int64_t)h * p.key_stride_head);
            load4<T>(src + e0, x);
            load4<T>(src + e1, y);
        }
        const void* weight = is_q ? p.q_weight : (is_v ? nullptr : p.key_weight);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = fmaf(x[i], x[i], fmaf(y[i], y[i], sum));
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (weight && live) {
            const float inv = 1.f / sqrtf(sum / (float)dim + p.eps);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] *= inv * (p.offset + weight_at(weight, p.weight_dtype, e0 + i));
                y[i] *= inv * (p.offset + weight_at(weight, p.weight_dtype, e1 + i));
            }
        }
        if (turned && live) {
            const float2* turn = turns + tok * half + part * 4;
            if (p.interleaved) {
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float2 u = turn[i >> 1], v = turn[2 + (i >> 1)];
                    const float xa = x[i], ya = y[i];
                    x[i] = xa * u.x - x[i + 1] * u.y, x[i + 1] = x[i + 1] * u.x + xa * u.y;
                    y[i] = ya * v.x - y[i + 1] * v.y, y[i + 1] = y[i + 1] * v.x + ya * v.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 u = turn[i];
                    const float xa = x[i];
                    x[i] = xa * u.x - y[i] * u.y, y[i] = y[i] * u.x + xa * u.y;
                }
            }
        }
        T* out = is_q ? (T*)p.q_out : (is_v ? nullptr : (T*)p.keys_out);
        if (out && live) {
            out += t * (is_q ? p.q_out_stride_token : p.key_out_stride_token) + (int64_t)h * (is_q ? p.q_out_stride_head : p.key_out_stride_head);
            store4<T>(out + e0, x);
            store4<T>(out + e1, y);
        }
        if constexpr (WRITE) {
            if (__all_sync(0xffffffffu, is_q || !here)) continue;
            // the row as eight neighbouring elements a lane, and into its page
            if (live && !is_q) {
#pragma unroll
                for (int i = 0; i < 4; ++i) relay[e0 + i] = x[i], relay[e1 + i] = y[i];
            }
            __syncwarp();
            float z[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = live && !is_q ? relay[part * 8 + i] : 0.f;
            __syncwarp();
            const int64_t slot = here && !is_q ? a.slots[t] : -1;
            const bool outside = slot >= 0 && a.slots_total && slot >= a.slots_total;
            if (outside && part == 0 && a.status) atomicExch(a.status, CRIT_B200_STATUS_BOUNDS);
            encode_row(a, z, live && slot >= 0 && !outside, is_v, slot, h, dim, part, LANES);
        }
    }
}

typedef void (*norm_rope_fn)(const crit_b200_norm_rope_params, const crit_b200_append_params, const int);

template <typename T, bool WRITE>
static norm_rope_fn norm_rope_lanes(int width) {
    if (width <= 64) return norm_rope_kernel<T, 8, WRITE>;
    if (width <= 128) return norm_rope_kernel<T, 16, WRITE>;
    return norm_rope_kernel<T, 32, WRITE>;
}

template <typename T>
static norm_rope_fn norm_rope_pick(int width, bool write) { return write ? norm_rope_lanes<T, true>(width) : norm_rope_lanes<T, false>(width); }

int check_append(const crit_b200_append_params& p);                                       // append.cu

}  // namespace crit_b200

using namespace crit_b200;

extern "C" __attribute__((visibility("default"))) int crit_b200_norm_rope(const crit_b200_norm_rope_params* params, const crit_b200_append_params* append,
                                                                          void* stream) {
    if (!params) return CRIT_B200_EINVAL;
    const crit_b200_norm_rope_params p = *params;
    if (p.tokens == 0) return 0;
    if (p.tokens < 0 || !p.positions || !p.frequencies || p.n_axes < 1 || (p.n_axes > 1 && !p.axes) || p.q_heads < 0 || p.kv_heads < 0 ||
        p.q_heads + p.kv_heads < 1 || (p.q_heads && (!p.q || !p.q_out)) || (p.kv_heads && (!p.keys || (!p.keys_out && !append))))
        return CRIT_B200_EINVAL;
    if (p.head_dim < 32 || p.head_dim > 256 || p.head_dim % 32 || p.rotary < 8 || p.rotary > p.head_dim || p.rotary % 8) return CRIT_B200_EUNSUPPORTED;
    if (p.dtype < 0 || p.dtype > CRIT_B200_DTYPE_FP32 || p.weight_dtype < 0 || p.weight_dtype > CRIT_B200_DTYPE_FP32) return CRIT_B200_EINVAL;
    const size_t vector = p.dtype == CRIT_B200_DTYPE_FP32 ? 16 : 8;
    const int64_t strides = (p.q_heads ? p.q_stride_token | p.q_stride_head | p.q_out_stride_token | p.q_out_stride_head : 0) |
                            (p.kv_heads ? p.key_stride_token | p.key_stride_head : 0) | (p.keys_out ? p.key_out_stride_token | p.key_out_stride_head : 0);
    if (strides % 4 || !aligned(p.q, vector) || !aligned(p.q_out, vector) || !aligned(p.keys, vector) || !aligned(p.keys_out, vector)) return CRIT_B200_EALIGN;
    crit_b200_append_params a;
    memset(&a, 0, sizeof a);
    int width = p.head_dim;
    if (append) {
        a = *append;
        a.keys = p.keys, a.key_stride_token = p.key_stride_token, a.key_stride_head = p.key_stride_head;
        if (a.tokens != p.tokens || a.kv_heads != p.kv_heads || a.head_dim != p.head_dim || a.in_dtype != p.dtype) return CRIT_B200_EINVAL;
        if (a.kind == CRIT_B200_KIND_FP8_PAGE) return CRIT_B200_EUNSUPPORTED;             // (a page's scale is its rows' together: two calls)
        if (int e = check_append(a)) return e;
        if (!aligned(a.key_pages, 16)) return CRIT_B200_EALIGN;
        if (a.values) {
            if ((a.value_stride_token | a.value_stride_head) % 4 || !aligned(a.values, vector) || !aligned(a.value_pages, 16)) return CRIT_B200_EALIGN;
            width = a.value_dim > width ? a.value_dim : width;
        }
    }
    const int row_heads = p.q_heads + p.kv_heads + (a.values ? p.kv_heads : 0);
    int per_block = 32 / row_heads;                                                        // a few rows a warp at least
    per_block = per_block < 1 ? 1 : (per_block > ROPE_MAX_TOKENS ? ROPE_MAX_TOKENS : per_block);
    const int lanes = width <= 64 ? 8 : (width <= 128 ? 16 : 32);
    const int smem = per_block * (p.rotary >> 1) * 8 + (append ? ROPE_WARPS * (32 / lanes) * (lanes * 8 + 4) * 4 : 0);
    const int64_t blocks = (p.tokens + per_block - 1) / per_block;
    if (blocks > 0x7fffffffLL) return CRIT_B200_EINVAL;
    norm_rope_fn fn;
    if (p.dtype == CRIT_B200_DTYPE_BF16) fn = norm_rope_pick<__nv_bfloat16>(width, append != nullptr);
    else if (p.dtype == CRIT_B200_DTYPE_FP16) fn = norm_rope_pick<__half>(width, append != nullptr);
    else fn = norm_rope_pick<float>(width, append != nullptr);
    fn<<<(unsigned)blocks, ROPE_WARPS * 32, smem, (cudaStream_t)stream>>>(p, a, per_block);
    CRIT_CHECK_LAUNCH();
    return 0;
}
