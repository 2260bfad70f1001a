// Split-K decode / speculative-verify attention over 4-bit pages (int4.cuh has the format).
//
// A block is a producer warp and a warp for each of HB kv heads (HB = 8, 4, 2 or 1: the most that divides the heads); it
// reads whole page rows, 16 positions of its HB heads a tile: one box of a tensor map with permuted dimensions, [dim / 2
// bytes][slots][kv_heads], is HB * dim / 2 contiguous bytes a position and lands head-major, swizzled as wide as a row is.
// So the bytes asked of HBM are long pieces although a row of one head is 64 bytes (dim 128), and no warp spends
// instructions on copies.  The tile's scales come by a bulk copy onto the same mbarrier.
//
// A warp attends its own head's query rows (up to 8 NT: the columns of a verify window times the heads of the kv head's
// group) and never waits for another warp.  Scores and outputs are m16n8k16 products, positions or value columns on the
// instruction's 16 rows, query rows on its 8 columns:
//   S^T[16 positions][8 query rows] = K Q^T    one accumulator a group of 32: a group's scale is one number a position,
//                                              so x = sum over groups of scale[position][group] * S_group, in FP32
//   O^T[32 values][8 query rows] += V^T (P .* scale)     the values' scales multiply the probabilities, a group at a time
// The codes never pass through a thread one by one: ldmatrix hands a thread the 8 codes of a position and group that its
// fragments want (K), or, transposed, 4 codes each of two neighbouring positions (V), and a mask, an OR and an add make two
// FP16 numbers of two codes.  The head dimension is consumed in the order the nibbles come, the queries laid out to match.
//
// The queries become FP16 with an exponent of their own a row (the largest element between 2^13 and 2^14), so no bf16 query
// overflows or vanishes.  Weights are 2^(x - ref) with ref at most 2 (in the exponent) above the running maximum and never
// below it: a weight is at most 1, times a scale of at most 61,440 it stays an FP16 number, and the running reference moves
// only when a score passes it.  Sums are FP32.
#include <mutex>

#include "int4.cuh"
#include "tensor_map.cuh"

namespace crit_b200 {

constexpr int D4_MAX_STAGES = 8;

// The most kv heads a block takes: 8, or 4 where a warp's accumulators want more registers than 9 warps leave (a quarter of
// an SM holds 3 of 9 warps, 168 registers a thread, and 2 of 5).
constexpr __host__ __device__ int decode4_heads(int d, int nt) { return d == 256 || nt == 4 ? 4 : 8; }

struct Decode4Launch {
    int heads;              // kv heads a block takes (HB)
    int ctiles;             // tiles of 8 NT query rows a window row takes
    int stages;             // of the ring
    int stage_bytes;
};

// Two FP16 numbers (code - 8 each) from the nibbles 0 and 4 (or 1 and 5) of a word.
__device__ __forceinline__ uint32_t codes_low(uint32_t w) {
    uint32_t x = (w & 0x000f000fu) | 0x64006400u;                  // 1024 + n
    __half2 h = __hsub2(*reinterpret_cast<__half2*>(&x), __floats2half2_rn(1032.f, 1032.f));
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t codes_high(uint32_t w) {
    uint32_t x = (w & 0x00f000f0u) | 0x64006400u;                  // 1024 + 16 n
    __half2 h = __hfma2(*reinterpret_cast<__half2*>(&x), __floats2half2_rn(0.0625f, 0.0625f), __floats2half2_rn(-72.f, -72.f));
    return *reinterpret_cast<uint32_t*>(&h);
}

// A lane's scales: bytes [a, a', b, b'] of two positions (a, b) and two neighbouring groups -> FP16 pairs (a, b) and (a', b').
__device__ __forceinline__ void scale_pairs(uint32_t x, uint32_t& even, uint32_t& odd) {
    even = (x << 7) & 0x7f807f80u;
    odd = (x >> 1) & 0x7f807f80u;
}

__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b) {
    __half2 h = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&h);
}
// all ones in the halves that are not zero
__device__ __forceinline__ uint32_t nonzero2(uint32_t a) {
    return __hne2_mask(*reinterpret_cast<__half2*>(&a), __floats2half2_rn(0.f, 0.f));
}

// Byte offset of 16-byte chunk c (a group of 32 codes) of row `row` of a tile, rows of D / 2 bytes with TMA's swizzle of
// that width.
template <int D>
__device__ __forceinline__ int chunk4(int row, int c) {
    if constexpr (D == 256) return row * 128 + ((c ^ (row & 7)) << 4);
    else if constexpr (D == 128) return row * 64 + ((c ^ ((row >> 1) & 3)) << 4);
    else return row * 32 + ((c ^ ((row >> 2) & 1)) << 4);
}

// MASKS: draft trees, sliding windows and block lists (else a column sees every position up to its own).
template <int D, int NT, bool MASKS>
__global__ void __launch_bounds__(32 * (decode4_heads(D, NT) + 1)) decode4_kernel(const crit_b200_attend_params p, const Decode4Launch u,
                                                      const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int NG = D / 32;                // groups of a row
    constexpr int ROWS = 8 * NT;
    constexpr int TPI = 2;                    // tiles an iteration takes
    constexpr float AHEAD = 2.f;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    __shared__ __align__(8) uint64_t bars_mem[2 * D4_MAX_STAGES];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int G = p.q_heads / p.kv_heads;
    const int HB = u.heads;
    const uint32_t full = smem_addr(bars_mem), empty = full + D4_MAX_STAGES * 8;
    if (threadIdx.x == 0) {
        for (int s = 0; s < u.stages; ++s) mbar_init(full + s * 8, 1), mbar_init(empty + s * 8, HB);
        mbar_init_fence();
    }
    __syncthreads();

    // -- the unit --------------------------------------------------------------------------------------------------------
    const int r = blockIdx.z, split = blockIdx.x;
    const int hg = blockIdx.y / u.ctiles, ct = blockIdx.y - hg * u.ctiles;
    int count = p.counts ? p.counts[r] : p.columns;
    count = count > p.columns ? p.columns : count;
    if (count <= 0 || ct * ROWS >= count * G) return;
    const int64_t first = p.firsts[r];
    const bool context = (p.flags & CRIT_B200_ATTEND_CONTEXT) != 0;       // the positions before `first` only
    const int64_t L = context ? first : first + count;
    const int64_t begin = (int64_t)split * p.chunk;
    if (begin >= L) {
        // a row that holds no position (a context row at position 0): zeros and -inf, as the fold of no state gives
        if (L <= 0 && split == 0 && !(p.flags & CRIT_B200_ATTEND_PARTIALS) && warp < HB) {
            for (int rr = 0; rr < ROWS; ++rr) {
                const int flat = ct * ROWS + rr, col = flat / G;
                if (col >= count) break;
                const int64_t token = p.starts[r] + col, head = (hg * HB + warp) * G + flat - col * G;
                for (int c = lane; c < D; c += 32) reinterpret_cast<uint16_t*>(p.out)[token * p.out_stride_token + head * p.out_stride_head + c] = 0;
                if (lane == 0 && p.lse) p.lse[token * p.q_heads + head] = -INFINITY;
            }
        }
        return;
    }
    const int64_t end = begin + p.chunk < L ? begin + p.chunk : L;
    const int nsplit = (int)((L + p.chunk - 1) / p.chunk);
    const int tile0 = (int)(begin >> 4), ntiles = (int)((end - begin + 15) >> 4);
    const int code_bytes = HB * 16 * (D / 2);                              // a tile's keys, or its values
    const int scale_bytes = 16 * p.kv_heads * NG;
    const int row_scales = p.kv_heads * NG;                                // bytes of a position's scales

    bool dead = false;
    if (warp == HB) {
        // -- producer ------------------------------------------------------------------------------------------------------
        const int32_t* table = p.tables + (int64_t)p.rows[r] * p.table_stride;
        const uint32_t tiles_per_page = (uint32_t)p.page >> 4;
        const uint32_t pages_total = (uint32_t)(p.slots / p.page);
        int stage = 0;
        uint32_t phase = 0;
        int pgs = 0;
        bool outside = false;
        for (int i = 0; i < ntiles && !dead; ++i) {
            if ((i & 31) == 0) pgs = i + lane < ntiles ? table[(uint32_t)(tile0 + i + lane) / tiles_per_page] : 0;
            const uint32_t listed = (uint32_t)__shfl_sync(0xffffffffu, pgs, i & 31);
            outside |= listed >= pages_total;             // the tensor's last page is read instead; reported below
            if (lane == 0) {
                const uint32_t tile = (uint32_t)(tile0 + i);
                const uint32_t pg = listed < pages_total ? listed : pages_total - 1;
                const int64_t slot0 = (int64_t)pg * p.page + ((tile % tiles_per_page) << 4);
                dead = !mbar_wait(empty + stage * 8, phase ^ 1);
                if (!dead) {
                    const uint32_t bar = full + stage * 8, at = smem_addr(smem) + stage * u.stage_bytes;
                    mbar_expect_tx(bar, (uint32_t)(2 * code_bytes + 2 * scale_bytes));
                    tma_load_3d(at, &kmap, 0, (int)slot0, hg * HB, bar);
                    bulk_load(at + 2 * code_bytes, (const char*)p.key_scales + slot0 * row_scales, scale_bytes, bar);
                    tma_load_3d(at + code_bytes, &vmap, 0, (int)slot0, hg * HB, bar);
                    bulk_load(at + 2 * code_bytes + scale_bytes, (const char*)p.value_scales + slot0 * row_scales, scale_bytes, bar);
                }
            }
            dead = __any_sync(0xffffffffu, dead);
            if (++stage == u.stages) stage = 0, phase ^= 1;
        }
        if (outside && lane == 0 && p.status) atomicExch(p.status, CRIT_B200_STATUS_BOUNDS);
        if (__syncthreads_or(dead ? 1 : 0)) {
            // a copy or a reader never came: the copies in flight get a last bounded chance to land
            if (lane == 0) {
                for (int s = 0; s < u.stages; ++s) mbar_wait(full + s * 8, 0, 1000000ull);
                if (p.status) atomicExch(p.status, CRIT_B200_STATUS_TMA);
            }
        }
        return;
    }

    // -- a head's warp: its queries ----------------------------------------------------------------------------------------
    const int h = hg * HB + warp;
    const int start = p.starts[r];
    uint32_t qb[NT][NG][4];                    // pairs (0, 4), (1, 5), (2, 6), (3, 7) of elements 32 group + 8 t + ..
    float mul[NT][2];                          // scores of the lane's query rows (8 nt + 2 t + e) into base-2 logits
    int lastpos[NT][2];                        // the last position they see (-1: a padding row)
    unsigned long long seen[MASKS ? NT : 1][2];
    const bool tree = MASKS && p.parents != nullptr;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int flat = ct * ROWS + nt * 8 + g;
        const int col = flat / G, gq = flat - col * G;
        const bool live = col < count;
        float amax = 0.f;
        uint4 raw[NG];
#pragma unroll
        for (int k = 0; k < NG; ++k) {
            raw[k] = make_uint4(0, 0, 0, 0);
            if (live)
                raw[k] = *reinterpret_cast<const uint4*>((const char*)p.q + ((int64_t)(start + col) * p.q_stride_token +
                                                                             (int64_t)(h * G + gq) * p.q_stride_head + k * 32 + t * 8) * 2);
        }
        auto element = [&](int k, int i) {
            const uint32_t w = (&raw[k].x)[i >> 1];
            if (p.q_dtype == CRIT_B200_DTYPE_BF16) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
            return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w >> 16 : w)));
        };
#pragma unroll
        for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(element(k, i)));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        int e = (int)((__float_as_uint(amax) >> 23) & 255u) - 127 - 13;
        e = amax > 0.f ? (e < -110 ? -110 : (e > 110 ? 110 : e)) : 0;
        const float down = __int_as_float((127 - e) << 23);
#pragma unroll
        for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) qb[nt][k][j] = pack2<false>(element(k, j) * down, element(k, j + 4) * down);
        // the lane's columns are query rows 2 t and 2 t + 1: their exponents live with lanes g = 2 t and 2 t + 1
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int er = __shfl_sync(0xffffffffu, e, (2 * t + j) * 4);
            mul[nt][j] = p.scale * LOG2E * __int_as_float((127 + er) << 23);
            const int at = ct * ROWS + nt * 8 + 2 * t + j;
            const int c = at / G;
            lastpos[nt][j] = c < count ? (int)(context ? first - 1 : first + c) : -1;
            if constexpr (MASKS) {
                // of the window's own positions a column of a draft tree sees itself and its ancestors (bit = column)
                seen[nt][j] = 0ull;
                if (tree && c < count) {
                    const int32_t* par = p.parents + start;
                    int from = c;
                    for (int hops = 0; from >= 0 && from < count && hops <= count; ++hops) {
                        seen[nt][j] |= 1ull << from;
                        from = par[from];
                    }
                }
            }
        }
    }

    float acc[NG][2][NT][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int k = 0; k < NG; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[k][i >> 2][nt][i & 3] = 0.f;
        m_run[nt][0] = m_run[nt][1] = -INFINITY;
        l_run[nt][0] = l_run[nt][1] = 0.f;
    }

    const int first32 = (int)first;
    int stage = 0;
    uint32_t phase = 0;
    // ldmatrix rows: lanes 0-7 and 8-15 name positions 0-7 and 8-15 of chunk 2 i, lanes 16-31 the same of chunk 2 i + 1
    const int lrow = (lane & 7) + 8 * ((lane >> 3) & 1), lchunk = lane >> 4;
    for (int i = 0; i < ntiles; i += TPI) {
        const int have = ntiles - i < TPI ? ntiles - i : TPI;
        float x[TPI][NT][4];
        uint32_t base[TPI];
        int stages[TPI];
        bool masked = MASKS;
#pragma unroll
        for (int v = 0; v < TPI; ++v) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) x[v][nt][c] = v < have ? 0.f : -INFINITY;
            if (v >= have) continue;
            stages[v] = stage;
            base[v] = smem_addr(smem) + stage * u.stage_bytes;
            if (!__all_sync(0xffffffffu, mbar_wait(full + stage * 8, phase))) {
                dead = true;
                break;
            }
            if (++stage == u.stages) stage = 0, phase ^= 1;
            masked |= ((tile0 + i + v) << 4) + 16 > first32;
            // scores
            const uint32_t ktile = base[v] + warp * (16 * (D / 2));
            const unsigned char* ks = smem + (base[v] - smem_addr(smem)) + 2 * code_bytes + h * NG;
#pragma unroll
            for (int k = 0; k < NG; k += 2) {
                uint32_t w[4];
                ldmatrix_x4(w, ktile + chunk4<D>(lrow, k + lchunk));
                // the scales of positions g and g + 8, groups k and k + 1
                const uint32_t a = *reinterpret_cast<const uint16_t*>(ks + g * row_scales + k);
                const uint32_t b = *reinterpret_cast<const uint16_t*>(ks + (g + 8) * row_scales + k);
                uint32_t pair[2];
                scale_pairs(a | (b << 16), pair[0], pair[1]);
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const float2 s = __half22float2(*reinterpret_cast<__half2*>(&pair[o]));
                    const uint32_t lo = w[2 * o], hi = w[2 * o + 1];
                    const uint32_t a1[4] = {codes_low(lo), codes_low(hi), codes_high(lo), codes_high(hi)};
                    const uint32_t a2[4] = {codes_low(lo >> 8), codes_low(hi >> 8), codes_high(lo >> 8), codes_high(hi >> 8)};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float c[4] = {0.f, 0.f, 0.f, 0.f};
                        mma16816<false>(c, a1, qb[nt][k + o][0], qb[nt][k + o][1]);
                        mma16816<false>(c, a2, qb[nt][k + o][2], qb[nt][k + o][3]);
                        x[v][nt][0] = fmaf(c[0], s.x, x[v][nt][0]), x[v][nt][1] = fmaf(c[1], s.x, x[v][nt][1]);
                        x[v][nt][2] = fmaf(c[2], s.y, x[v][nt][2]), x[v][nt][3] = fmaf(c[3], s.y, x[v][nt][3]);
                    }
                }
            }
        }
        if (dead) break;

        // masks, online softmax
        uint32_t pb[TPI][NT][2];
        bool rescale = false;
        float alpha[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int v = 0; v < TPI; ++v)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float y = x[v][nt][c] * mul[nt][c & 1];
                    if (v >= have) y = -INFINITY;
                    if (masked) {
                        const int pos = ((tile0 + i + v) << 4) + g + 8 * (c >> 1), last = lastpos[nt][c & 1];
                        if (pos > last) y = -INFINITY;
                        if constexpr (MASKS) {
                            if (p.sliding > 0 && pos <= last - p.sliding) y = -INFINITY;
                            if (p.blocks && last >= 0) {
                                const int32_t* listed = p.blocks + (int64_t)(start + (last - first32)) * p.blocks_k;
                                const int block = pos / p.block_size;
                                bool member = false;
                                for (int j = 0; j < p.blocks_k; ++j) member |= listed[j] == block;
                                if (!member) y = -INFINITY;
                            }
                            if (tree && pos >= first32 && (pos - first32 >= count || !((seen[nt][c & 1] >> (pos - first32)) & 1ull)))
                                y = -INFINITY;
                        }
                    }
                    x[v][nt][c] = y;
                    mx[c & 1] = fmaxf(mx[c & 1], y);
                }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 4));
                mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 8));
                mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 16));
                const bool moved = mx[j] > m_run[nt][j];
                const float top = moved ? mx[j] + AHEAD : m_run[nt][j];
                const float sub = top == -INFINITY ? 0.f : top;
                alpha[nt][j] = moved ? ex2(m_run[nt][j] - sub) : 1.f;
                rescale |= moved;
                m_run[nt][j] = top;
                mx[j] = sub;
            }
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int v = 0; v < TPI; ++v) {
                float w[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    w[c] = ex2(x[v][nt][c] - mx[c & 1]);
                    sum[c & 1] += w[c];
                }
                pb[v][nt][0] = movmatrix_trans(pack2<false>(w[0], w[1]));
                pb[v][nt][1] = movmatrix_trans(pack2<false>(w[2], w[3]));
            }
            l_run[nt][0] = l_run[nt][0] * alpha[nt][0] + sum[0];
            l_run[nt][1] = l_run[nt][1] * alpha[nt][1] + sum[1];
        }
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
            for (int k = 0; k < NG; ++k)
#pragma unroll
                for (int o = 0; o < 2; ++o)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        acc[k][o][nt][0] *= alpha[nt][0], acc[k][o][nt][1] *= alpha[nt][1];
                        acc[k][o][nt][2] *= alpha[nt][0], acc[k][o][nt][3] *= alpha[nt][1];
                    }
        }

        // outputs
#pragma unroll
        for (int v = 0; v < TPI; ++v) {
            if (v >= have) continue;
            const uint32_t vtile = base[v] + code_bytes + warp * (16 * (D / 2));
            const unsigned char* vs = smem + (base[v] - smem_addr(smem)) + 2 * code_bytes + scale_bytes + h * NG;
            uint32_t keep[NT][2];                     // where a position is masked its scale may be anything, a NaN too
            if (masked) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) keep[nt][0] = nonzero2(pb[v][nt][0]), keep[nt][1] = nonzero2(pb[v][nt][1]);
            }
#pragma unroll
            for (int k = 0; k < NG; k += 2) {
                uint32_t w[4];
                ldmatrix_x4_trans(w, vtile + chunk4<D>(lrow, k + lchunk));
                // the scales of positions 2 t, 2 t + 1 and 2 t + 8, 2 t + 9, groups k and k + 1
                uint32_t pair[2][2];
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const uint32_t a = *reinterpret_cast<const uint16_t*>(vs + (2 * t + 8 * hf) * row_scales + k);
                    const uint32_t b = *reinterpret_cast<const uint16_t*>(vs + (2 * t + 1 + 8 * hf) * row_scales + k);
                    scale_pairs(a | (b << 16), pair[0][hf], pair[1][hf]);
                }
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const uint32_t lo = w[2 * o], hi = w[2 * o + 1];            // positions 0-7 and 8-15, values 4 g .. 4 g + 3
                    const uint32_t a1[4] = {codes_low(lo), codes_high(lo), codes_low(hi), codes_high(hi)};
                    const uint32_t a2[4] = {codes_low(lo >> 8), codes_high(lo >> 8), codes_low(hi >> 8), codes_high(hi >> 8)};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        uint32_t b0 = hmul2_bits(pb[v][nt][0], pair[o][0]), b1 = hmul2_bits(pb[v][nt][1], pair[o][1]);
                        if (masked) b0 &= keep[nt][0], b1 &= keep[nt][1];
                        mma16816<false>(acc[k + o][0][nt], a1, b0, b1);
                        mma16816<false>(acc[k + o][1][nt], a2, b0, b1);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(empty + stages[v] * 8) : "memory");
        }
    }
    if (__syncthreads_or(dead ? 1 : 0)) return;

    // -- the state, or the row's output --------------------------------------------------------------------------------------
    const bool whole = nsplit == 1 && !(p.flags & CRIT_B200_ATTEND_PARTIALS) && !p.sinks;     // (sinks join in the fold)
    const int64_t states = (int64_t)p.partial_rows * p.q_heads * p.max_splits;
    const int prow0 = p.offsets ? p.offsets[r] - p.offsets[0] : r * p.columns;
    const bool fits = whole || (p.workspace && split < p.max_splits && prow0 >= 0 && prow0 + count <= p.partial_rows);
    if (!fits) {
        if (lane == 0 && p.status) atomicExch(p.status, CRIT_B200_STATUS_PLAN);
        return;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float l = l_run[nt][j];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            const int flat = ct * ROWS + nt * 8 + 2 * t + j;
            const int col = flat / G, gq = flat - col * G;
            if (col >= count) continue;
            const int token = start + col, head = h * G + gq;
            if (whole) {
                const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);          // (a NaN stays one)
                char* dst = (char*)p.out + ((int64_t)token * p.out_stride_token + (int64_t)head * p.out_stride_head + 4 * g) * 2;
#pragma unroll
                for (int k = 0; k < NG; ++k) {
                    const float o0 = acc[k][0][nt][j] * inv, o1 = acc[k][0][nt][2 + j] * inv, o2 = acc[k][1][nt][j] * inv, o3 = acc[k][1][nt][2 + j] * inv;
                    *reinterpret_cast<uint2*>(dst + k * 64) =
                        p.q_dtype == CRIT_B200_DTYPE_BF16 ? make_uint2(pack2<true>(o0, o1), pack2<true>(o2, o3)) : make_uint2(pack2<false>(o0, o1), pack2<false>(o2, o3));
                }
                if (p.lse && g == 0) p.lse[(int64_t)token * p.q_heads + head] = l == 0.f ? -INFINITY : m_run[nt][j] * LN2 + logf(l);
            } else {
                const int64_t at = ((int64_t)(prow0 + col) * p.q_heads + head) * p.max_splits + split;
                float* dst = p.workspace + at * D + 4 * g;
#pragma unroll
                for (int k = 0; k < NG; ++k)
                    *reinterpret_cast<float4*>(dst + k * 32) = make_float4(acc[k][0][nt][j], acc[k][0][nt][2 + j], acc[k][1][nt][j], acc[k][1][nt][2 + j]);
                if (g == 0) {
                    p.workspace[states * D + at] = m_run[nt][j];
                    p.workspace[states * (D + 1) + at] = l;
                }
            }
        }
}

// -- host side --------------------------------------------------------------------------------------------------------------
typedef void (*decode4_fn)(const crit_b200_attend_params, const Decode4Launch, const CUtensorMap, const CUtensorMap);

template <int D, int NT>
static decode4_fn decode4_of(bool masks) {
    if (masks) return decode4_kernel<D, NT, true>;
    return decode4_kernel<D, NT, false>;
}

static decode4_fn decode4_pick(int d, int nt, bool masks) {
    switch (d) {
        case 64: return nt == 1 ? decode4_of<64, 1>(masks) : (nt == 2 ? decode4_of<64, 2>(masks) : decode4_of<64, 4>(masks));
        case 128: return nt == 1 ? decode4_of<128, 1>(masks) : (nt == 2 ? decode4_of<128, 2>(masks) : decode4_of<128, 4>(masks));
        case 256: return nt == 1 ? decode4_of<256, 1>(masks) : decode4_of<256, 2>(masks);
        default: return nullptr;
    }
}

static int heads_of(int kv_heads, int most) {
    int heads = most;
    while (kv_heads % heads) heads >>= 1;
    return heads;
}

// The launch of a geometry: query-row tiles, heads a block takes, stages that two blocks' shares of an SM hold.
static int decode4_shape(int q_heads, int kv_heads, int d, int columns, int* nt, Decode4Launch* u, int* smem) {
    if (d != 64 && d != 128 && d != 256) return CRIT_B200_EUNSUPPORTED;
    const int rows = columns * (q_heads / kv_heads);
    *nt = rows <= 8 ? 1 : (rows <= 16 || d == 256 ? 2 : 4);
    u->heads = heads_of(kv_heads, decode4_heads(d, *nt));
    u->ctiles = (rows + 8 * *nt - 1) / (8 * *nt);
    u->stage_bytes = (u->heads * 16 * d + 2 * 16 * kv_heads * (d / 32) + 1023) / 1024 * 1024;
    const int want = 16 * 1024 * u->heads;                                    // in flight a block: 128 KB for 8 heads
    const int room = 110 * 1024;
    int stages = (want < room ? want : room) / u->stage_bytes;
    u->stages = stages < 2 ? 2 : (stages > D4_MAX_STAGES ? D4_MAX_STAGES : stages);
    *smem = 1024 + u->stages * u->stage_bytes;
    return *smem > 226 * 1024 ? CRIT_B200_EUNSUPPORTED : 0;
}

int launch_decode4(const crit_b200_attend_params& p, cudaStream_t s) {
    if (p.flags & (CRIT_B200_ATTEND_TCGEN05 | CRIT_B200_ATTEND_TCGEN05P | CRIT_B200_ATTEND_TCGEN05T)) return CRIT_B200_EUNSUPPORTED;
    if (p.head_dim != p.value_dim || p.slots < 16 || p.slots > 0x7fffffffLL || p.slots < p.page) return CRIT_B200_EUNSUPPORTED;
    if (!aligned(p.key_scales, 16) || !aligned(p.value_scales, 16)) return CRIT_B200_EALIGN;
    int nt = 0, smem = 0;
    Decode4Launch u;
    if (int e = decode4_shape(p.q_heads, p.kv_heads, p.head_dim, p.columns, &nt, &u, &smem)) return e;
    CUtensorMap kmap, vmap;
    if (!rows4_map(&kmap, p.key_pages, p.head_dim, p.kv_heads, u.heads, p.slots) ||
        !rows4_map(&vmap, p.value_pages, p.head_dim, p.kv_heads, u.heads, p.slots))
        return CRIT_B200_EUNSUPPORTED;
    const decode4_fn fn = decode4_pick(p.head_dim, nt, p.parents || p.sliding > 0 || p.blocks);
    cudaError_t ce = cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (ce != cudaSuccess) return (int)ce;
    const int64_t hg = p.kv_heads / u.heads;
    if (hg * u.ctiles > 65535 || p.n_rows > 65535) return CRIT_B200_EUNSUPPORTED;
    dim3 grid((unsigned)p.max_splits, (unsigned)(hg * u.ctiles), (unsigned)p.n_rows);
    fn<<<grid, 32 * (u.heads + 1), smem, s>>>(p, u, kmap, vmap);
    CRIT_CHECK_LAUNCH();
    return 0;
}

int plan_decode4(int q_heads, int kv_heads, int d, int columns, int32_t* out5) {
    int nt = 0, smem = 0, device = 0, sms = 0, per_sm = 0;
    Decode4Launch u;
    if (int e = decode4_shape(q_heads, kv_heads, d, columns, &nt, &u, &smem)) return e;
    const decode4_fn fn = decode4_pick(d, nt, false);
    if (cudaGetDevice(&device) == cudaSuccess) {
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        if (cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess)
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, (const void*)fn, 32 * (u.heads + 1), smem);
    }
    cudaGetLastError();
    out5[0] = 1024, out5[1] = smem, out5[2] = 8 * nt, out5[3] = per_sm, out5[4] = sms;
    return 0;
}

}  // namespace crit_b200
