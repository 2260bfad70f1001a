// The step in front of the cache: each head of the queries and keys divided by its root mean square and weighted, its pairs
// turned by angles of the token's position(s), and (when the call writes) the keys and values encoded into their pages, in
// one launch.
//
//   y = x / sqrt(mean x^2 + eps) * (offset + w)                              where a weight is given, else y = x
//   (a, b) -> magnitude * (a cos - b sin, b cos + a sin)                     pairs (i, rotary / 2 + i), or (2 i, 2 i + 1)
//   angle of pair i = positions[axes[i]][token] * frequencies[i]             (axes NULL: positions[token])
//
// A warp takes a token's heads, or a part of them where there are too few tokens to fill the device: it makes the sines and
// cosines once (32 lanes, two pairs each of a rotation of 128; the angle is a product in FP64, since a position of 2^20 times
// a frequency loses 2^-4 of a radian in FP32, reduced to a part of a turn there and handed to sincospi in FP32, what FP32 leaves of it put back after), multiplies
// the head weights into them, and walks the queries' rows, the keys' and (when it writes) the values'.  8, 16 or 32 lanes
// share a row of up to 64, 128 or 256 elements: a lane holds four pairs, two vectors of four elements, so nothing crosses
// lanes but the sum of squares, and a row is in flight while the one before it is worked on.  A row that goes to a page is
// laid out again through shared memory, eight neighbouring elements a lane, and encoded from its FP32 values as
// crit_b200_append encodes rows (16-bit pages, E4M3, INT8 and 4-bit codes).
// All sums are FP32; a result is rounded once.  Every element is read and written once.
// Measured: 8,192 tokens of 32 + 8 heads of 128, bf16: 35.9 us, 168 MB at 4.7 TB/s (floor 25.6 us); keys and values to 4-bit pages
// in the same pass: 46.6 us for 177 MB (floor 27), bound by the codes' instructions (70% of the issue slots full; the values at 8
// elements a lane 50 us, the keys at 16 by way of two turns' rows in shared memory no faster); a step of 64 tokens of 64 + 8 heads:
// 4.1 us, with the append 4.8, the launch and one row's latency.
#include <type_traits>

#include "int4.cuh"

namespace crit_b200 {

constexpr int ROPE_WARPS = 8;
// Warps an SM that a launch of few tokens is to have: a token's heads are dealt to more warps until then, each of which makes the
// token's sines again.  8,192 tokens with the append and two reads back: 65 us with 32 (and 16), 75 with 64; 64 tokens: 8.6 us
// with 32, 9.3 with 16.
constexpr int ROPE_FILL = 32;

template <typename T>
__device__ __forceinline__ void store4(T* dst, const float (&x)[4]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]));
    }
}

// A lane's eight neighbouring elements of a row (lane `part` of the row's lanes, `span` of them) into the row's page slot.
// Every lane of the warp comes here: lanes without elements (or whose row is not written) with live false.
__device__ __forceinline__ void encode_row(const crit_b200_append_params& a, float (&x)[8], bool live, bool is_v, int64_t slot, int h,
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

// Four elements as they lie in memory, and as FP32.
template <typename T>
struct Raw4 {
    typename std::conditional<sizeof(T) == 4, float4, uint2>::type v;
    __device__ __forceinline__ void load(const T* src) { v = *reinterpret_cast<const decltype(v)*>(src); }
    __device__ __forceinline__ void floats(float (&x)[4]) const {
        if constexpr (sizeof(T) == 4) {
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
            x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
        } else {
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
            x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
        }
    }
};

// offset + a weight's four elements from e.
__device__ __forceinline__ void weight4(const void* weight, int dtype, int e, float offset, float (&w)[4]) {
    if (dtype == CRIT_B200_DTYPE_FP32) {
        const float* at = (const float*)weight + e;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = at[i];
    } else {
        const uint16_t* at = (const uint16_t*)weight + e;
        uint2 v;
        if ((reinterpret_cast<uintptr_t>(at) & 7) == 0) v = *reinterpret_cast<const uint2*>(at);
        else v = make_uint2(at[0] | ((uint32_t)at[1] << 16), at[2] | ((uint32_t)at[3] << 16));
        if (dtype == CRIT_B200_DTYPE_BF16) {
            Raw4<__nv_bfloat16> raw;
            raw.v = v, raw.floats(w);
        } else {
            Raw4<__half> raw;
            raw.v = v, raw.floats(w);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] += offset;
}

// LANES: of a row (8, 16 or 32: the widest head has up to 8 elements a lane).  NEIGHBOURS: pairs (2 i, 2 i + 1).  parts: warps that
// share a token.
template <typename T, int LANES, bool WRITE, bool NEIGHBOURS>
__global__ void __launch_bounds__(ROPE_WARPS * 32, 4) norm_rope_kernel(const crit_b200_norm_rope_params p, const crit_b200_append_params a, const int parts,
                                                                    const float inv_dim) {
    constexpr int ROWS = 32 / LANES;                         // rows a warp holds at once
    constexpr int DEPTH = 3;                                 // rows in flight: 8,192 tokens 37.6 us, with 2 39.5, 4 slower too
    __shared__ __align__(16) float2 turns_mem[ROPE_WARPS][128];            // (cos, sin) of the warp's token
    __shared__ __align__(16) float relay_mem[WRITE ? ROPE_WARPS * ROWS : 1][WRITE ? LANES * 8 + 4 : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane % LANES, sub = lane / LANES;
    const int64_t job = (int64_t)blockIdx.x * ROPE_WARPS + warp;
    const int64_t t = job / parts;
    if (t >= p.tokens) return;                               // (no barrier of the block follows)
    const int piece = (int)(job - t * parts);
    const int half = p.rotary >> 1;
    float2* turns = turns_mem[warp];

    // the lane's two vectors of four elements in a row: of a turned chunk the pairs' halves (or four neighbouring pairs), of
    // the rest eight neighbours
    const bool turned = part * 4 < half;
    const int e0 = turned ? (NEIGHBOURS ? part * 8 : part * 4) : p.rotary + (part - (half >> 2)) * 8;
    const int e1 = turned && !NEIGHBOURS ? half + part * 4 : e0 + 4;
    const bool inside = part * 8 < p.head_dim;

    // this warp's share of the token's rows, the queries' first, then the keys', then the values'
    const int row_heads = p.q_heads + p.kv_heads + (WRITE && a.values ? p.kv_heads : 0);
    const int share = (row_heads + parts - 1) / parts, begin = piece * share, end = begin + share;
    const int q0 = begin < p.q_heads ? begin : p.q_heads, q1 = end < p.q_heads ? end : p.q_heads;
    auto within = [&](int x) { x -= p.q_heads; return x < 0 ? 0 : (x > p.kv_heads ? p.kv_heads : x); };
    const int k0 = within(begin), k1 = within(end), v0 = within(begin - p.kv_heads), v1 = WRITE && a.values ? within(end - p.kv_heads) : 0;

    // Rows on their way from memory: DEPTH of them ahead of the one that is worked on (h + d ROWS + sub is a lane's row).
    Raw4<T> ra[DEPTH], rb[DEPTH];
    auto ask = [&](const T* rows, int64_t stride, int row, int upto, int d) {
        if (inside && row < upto) ra[d].load(rows + row * stride + e0), rb[d].load(rows + row * stride + e1);
    };
    const T* q_rows = (const T*)p.q + t * p.q_stride_token;
    const T* k_rows = (const T*)p.keys + t * p.key_stride_token;
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) ask(q_rows, p.q_stride_head, q0 + d * ROWS + sub, q1, d);           // (before the sines are made)

    for (int pair = lane; pair < half; pair += 32) {
        const int axis = p.axes ? p.axes[pair] : 0;
        float2 turn = make_float2(0.f, 0.f);
        if (axis >= 0 && axis < p.n_axes) {
            const double at = (double)p.positions[(int64_t)axis * p.axis_stride + t] * (double)p.frequencies[pair];
            // at / (2 pi) less its whole turns: 1 / (2 pi) as a sum of two FP64 numbers, the product's rounding put back
            const double turns_of = at * 0.15915494309189535;
            const double rest = fma(at, 0.15915494309189535, -turns_of) + at * -9.839338337591243e-18;
            const double halves = 2.0 * ((turns_of - rint(turns_of)) + rest);
            const float near = (float)halves, beside = (float)(halves - (double)near) * 3.14159265f;      // what FP32 leaves of the angle, in radians
            float s, c;
            sincospif(near, &s, &c);
            turn = make_float2(fmaf(-s, beside, c) * p.magnitude, fmaf(c, beside, s) * p.magnitude);
        } else if (p.status) {
            atomicExch(p.status, CRIT_B200_STATUS_BOUNDS);   // an axis that positions has not: the pair becomes zeros
        }
        turns[pair] = turn;
    }
    __syncwarp();

    // A result is an element and its partner times two factors: the first vector's own and partner's, the second's own and
    // partner's (cos and sin with the head's weights; 1 and 0 past the rotation).
    float own0[4], other0[4], own1[4], other1[4];
    auto factors = [&](const void* weight) {
        float w0[4] = {1.f, 1.f, 1.f, 1.f}, w1[4] = {1.f, 1.f, 1.f, 1.f};
        if (weight && inside) weight4(weight, p.weight_dtype, e0, p.offset, w0), weight4(weight, p.weight_dtype, e1, p.offset, w1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!turned) {
                own0[i] = w0[i], own1[i] = w1[i], other0[i] = other1[i] = 0.f;
            } else if (NEIGHBOURS) {
                const float2 u = turns[part * 4 + (i >> 1)], v = turns[part * 4 + 2 + (i >> 1)];
                own0[i] = u.x * w0[i], other0[i] = (i & 1 ? u.y : -u.y) * w0[i ^ 1];
                own1[i] = v.x * w1[i], other1[i] = (i & 1 ? v.y : -v.y) * w1[i ^ 1];
            } else {
                const float2 u = turns[part * 4 + i];
                own0[i] = u.x * w0[i], other0[i] = -u.y * w1[i];
                own1[i] = u.x * w1[i], other1[i] = u.y * w0[i];
            }
        }
    };
    auto turn_row = [&](float (&x)[4], float (&y)[4], bool normed) {
        float inv = 1.f;
        if (normed) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum = fmaf(x[i], x[i], fmaf(y[i], y[i], sum));
#pragma unroll
            for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            inv = rsqrtf(fmaf(sum, inv_dim, p.eps));
        }
        float u[4], v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float partner0 = NEIGHBOURS ? x[i ^ 1] : y[i], partner1 = NEIGHBOURS ? y[i ^ 1] : x[i];
            u[i] = fmaf(partner0, other0[i], x[i] * own0[i]) * inv, v[i] = fmaf(partner1, other1[i], y[i] * own1[i]) * inv;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = u[i], y[i] = v[i];
    };

    // -- the queries' rows --------------------------------------------------------------------------------------------------
    if (q0 < q1) {
        factors(p.q_weight);
        T* out = (T*)p.q_out + t * p.q_out_stride_token;
        for (int h0 = q0; h0 < q1; h0 += ROWS * DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int h = h0 + d * ROWS;                 // (the same for every lane)
                if (h >= q1) break;
                float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
                const bool live = inside && h + sub < q1;
                if (live) ra[d].floats(x), rb[d].floats(y);
                ask(q_rows, p.q_stride_head, h + DEPTH * ROWS + sub, q1, d);
                turn_row(x, y, p.q_weight != nullptr);
                if (live) {
                    T* to = out + (h + sub) * p.q_out_stride_head;
                    store4<T>(to + e0, x), store4<T>(to + e1, y);
                }
            }
        }
    }

    // -- the keys' rows, and their pages -------------------------------------------------------------------------------------
    int64_t slot = -1;
    if (WRITE && (k0 < k1 || v0 < v1)) {
        slot = a.slots[t];
        if (slot >= 0 && a.slots_total && slot >= a.slots_total) {       // outside the page tensor: skipped and reported
            if (lane == 0 && a.status) atomicExch(a.status, CRIT_B200_STATUS_BOUNDS);
            slot = -1;
        }
    }
    if (k0 < k1) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) ask(k_rows, p.key_stride_head, k0 + d * ROWS + sub, k1, d);
        factors(p.key_weight);
        T* out = p.keys_out ? (T*)p.keys_out + t * p.key_out_stride_token : nullptr;
        for (int h0 = k0; h0 < k1; h0 += ROWS * DEPTH) {
#pragma unroll
          for (int d = 0; d < DEPTH; ++d) {
            const int h = h0 + d * ROWS;
            if (h >= k1) break;
            float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
            const bool live = inside && h + sub < k1;
            if (live) ra[d].floats(x), rb[d].floats(y);
            ask(k_rows, p.key_stride_head, h + DEPTH * ROWS + sub, k1, d);
            turn_row(x, y, p.key_weight != nullptr);
            if (out && live) {
                T* to = out + (h + sub) * p.key_out_stride_head;
                store4<T>(to + e0, x), store4<T>(to + e1, y);
            }
            if constexpr (WRITE) {
                if (slot < 0) continue;                      // (the warp's token: the same for every lane)
                float* relay = relay_mem[warp * ROWS + sub];  // the row as eight neighbouring elements a lane
                if (live) {
                    *reinterpret_cast<float4*>(relay + e0) = make_float4(x[0], x[1], x[2], x[3]);
                    *reinterpret_cast<float4*>(relay + e1) = make_float4(y[0], y[1], y[2], y[3]);
                }
                __syncwarp();
                float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (live) {
                    const float4 u = *reinterpret_cast<const float4*>(relay + part * 8), v = *reinterpret_cast<const float4*>(relay + part * 8 + 4);
                    z[0] = u.x, z[1] = u.y, z[2] = u.z, z[3] = u.w, z[4] = v.x, z[5] = v.y, z[6] = v.z, z[7] = v.w;
                }
                __syncwarp();
                encode_row(a, z, live, false, slot, h + sub, p.head_dim, part, LANES);
            }
          }
        }
    }

    // -- the values' rows go to their pages as they are ----------------------------------------------------------------------
    if (WRITE && v0 < v1 && slot >= 0 && a.kind == CRIT_B200_KIND_INT4) {       // 16 elements a lane, as crit_b200_append takes them
        const int vpart = lane % (LANES / 2), vsub = lane / (LANES / 2);
        const bool held = vpart * 16 < a.value_dim;
        const T* v_row = (const T*)a.values + t * a.value_stride_token + (int64_t)(v0 + vsub) * a.value_stride_head + vpart * 16;
        for (int h = v0; h < v1; h += 2 * ROWS) {
            float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            const bool live = held && h + vsub < v1;
            if (live) {
                Raw4<T> v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i].load(v_row + 4 * i);
                v[0].floats(reinterpret_cast<float(&)[4]>(y[0])), v[1].floats(reinterpret_cast<float(&)[4]>(y[4]));
                v[2].floats(reinterpret_cast<float(&)[4]>(z[0])), v[3].floats(reinterpret_cast<float(&)[4]>(z[4]));
            }
            v_row += 2 * ROWS * a.value_stride_head;
            int bits = max(int4_top(y), int4_top(z));
            bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
            const uint32_t byte = int4_scale_byte(__int_as_float(bits), bits > 0x7f800000);
            const float s = int4_scale(byte);
            const uint2 w = make_uint2(int4_codes(y, s, byte), int4_codes(z, s, byte));
            if (!live) continue;
            const int64_t row = slot * a.kv_heads + h + vsub;
            reinterpret_cast<uint2*>(a.value_pages)[row * (a.value_dim >> 4) + vpart] = w;
            if ((vpart & 1) == 0) reinterpret_cast<uint8_t*>(a.value_scales)[row * (a.value_dim >> 5) + (vpart >> 1)] = (uint8_t)byte;
        }
    } else if (WRITE && v0 < v1 && slot >= 0) {
        const bool held = part * 8 < a.value_dim;
        const T* v_row = (const T*)a.values + t * a.value_stride_token + (int64_t)(v0 + sub) * a.value_stride_head + part * 8;
        for (int h = v0; h < v1; h += ROWS) {
            float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            const bool live = held && h + sub < v1;
            if (live) {
                Raw4<T> va, vb;
                va.load(v_row), vb.load(v_row + 4);
                va.floats(reinterpret_cast<float(&)[4]>(z[0])), vb.floats(reinterpret_cast<float(&)[4]>(z[4]));
            }
            v_row += ROWS * a.value_stride_head;
            encode_row(a, z, live, true, slot, h + sub, a.value_dim, part, LANES);
        }
    }
}

typedef void (*norm_rope_fn)(const crit_b200_norm_rope_params, const crit_b200_append_params, const int, const float);

template <typename T, int LANES>
static norm_rope_fn norm_rope_of(bool write, bool neighbours) {
    if (write) return neighbours ? norm_rope_kernel<T, LANES, true, true> : norm_rope_kernel<T, LANES, true, false>;
    return neighbours ? norm_rope_kernel<T, LANES, false, true> : norm_rope_kernel<T, LANES, false, false>;
}

template <typename T>
static norm_rope_fn norm_rope_pick(int width, bool write, bool neighbours) {
    if (width <= 64) return norm_rope_of<T, 8>(write, neighbours);
    return width <= 128 ? norm_rope_of<T, 16>(write, neighbours) : norm_rope_of<T, 32>(write, neighbours);
}

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
    // Warps a token: one for a prompt of many tokens (a token's sines are made once), as many as it has rows for a step's few,
    // so that the launch fills the device once or a warp has one iteration.
    const int row_heads = p.q_heads + p.kv_heads + (a.values ? p.kv_heads : 0);
    const int rows_at_once = 32 / (width <= 64 ? 8 : (width <= 128 ? 16 : 32)), most = (row_heads + rows_at_once - 1) / rows_at_once;
    int device = 0, sms = 0;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) sms = 1;
    const int64_t wanted = ((int64_t)sms * ROPE_FILL + p.tokens - 1) / p.tokens;
    const int parts = (int)(wanted < most ? wanted : most);
    const int64_t blocks = (p.tokens * parts + ROPE_WARPS - 1) / ROPE_WARPS;
    if (blocks > 0x7fffffffLL) return CRIT_B200_EINVAL;
    norm_rope_fn fn;
    if (p.dtype == CRIT_B200_DTYPE_BF16) fn = norm_rope_pick<__nv_bfloat16>(width, append != nullptr, p.interleaved != 0);
    else if (p.dtype == CRIT_B200_DTYPE_FP16) fn = norm_rope_pick<__half>(width, append != nullptr, p.interleaved != 0);
    else fn = norm_rope_pick<float>(width, append != nullptr, p.interleaved != 0);
    fn<<<(unsigned)blocks, ROPE_WARPS * 32, 0, (cudaStream_t)stream>>>(p, a, parts, 1.f / (float)p.head_dim);
    CRIT_CHECK_LAUNCH();
    return 0;
}
