// Split-K decode / speculative-verify attention over 4-bit pages (int4.cuh has the format).
//
// A block is a warp for each of HB kv heads (8, 4, 2 or 1: the most that divides the heads) and reads whole page rows, 16
// positions of its HB heads a tile: one box of a tensor map with permuted dimensions, [128 bytes][slots][rows of 128 a slot], is
// HB * dim / 2 contiguous bytes a position and lands with a few heads' (two of dim 128) 16 positions together, swizzled.  So the
// bytes asked of HBM are long pieces although a row of one head is 64 bytes (dim 128).  The tile's scales come by a
// bulk copy onto the same mbarrier.  There is no producer warp (a ninth warp would take the registers of two blocks an SM): the
// warps take turns, warp n mod HB refills the ring when it comes to tile n, with a tile S - 3 ahead and the page id it read
// a turn before.
//
// A warp attends its own head's query rows (up to 8 NT: the columns of a verify window times the heads of the kv head's
// group) and waits for the others only through the ring.  Scores and outputs are m16n8k16 products, positions or value
// columns on the instruction's 16 rows, query rows on its 8 columns:
//   S^T[16 positions][8 query rows] = K Q^T    one accumulator a group of 32: a group's scale is one number a position,
//                                              so x = sum over groups of scale[position][group] * S_group, in FP32
//   O^T[32 values][8 query rows] += V^T P^T    the values' scales multiply the codes
// The codes never pass through a thread one by one: ldmatrix hands a thread the 8 codes of a position and group that its
// fragments want (K), or, transposed, 4 codes each of two neighbouring positions (V).  The head dimension is consumed in the
// order the nibbles come, the queries laid out to match.
//
// Codes as FP16 operands.  The nibbles 0 and 4 of a word under the mask 0x000f000f ARE two FP16 numbers, n * 2^-24 (subnormal;
// the tensor cores take them as they are), the nibbles 1 and 5 under 0x00f000f0 are 16 n * 2^-24: one AND makes two operands,
// where 1024 + n less 1032 takes an OR and an add more.  The keys are taken so: the factor 16 is undone in the queries (their
// odd elements are divided by 16), 2^-24 in a constant, and the 8 that a code stands above its value comes off in a product of
// its own, the positions' scales with -8 * the sums of the groups' queries (a K of the groups' number, the sums as two FP16
// terms).  Where the accumulators for that do not fit the registers (wide tiles of query rows), codes become n - 8 one add
// later.  The values become (n - 8) * s with s the scale over 128, exactly: 8 significant bits, from 2^-24 up to 3,840.  The
// nibbles 1 and 5 in one FMA: under 0x5400 they are 64 + n, and (64 + n) * s - 72 * s has no rounding (72 * s: 8 bits too); the
// nibbles 0 and 4 as n - 8, then times s.  (All of them by the FMA take more shifts, which wait for the integer pipe: 64 rows of
// 4,096 88.3 us against 86.8; all of them as n - 8 first 88.1.)
//
// The queries become FP16 with an exponent of their own a row (the largest element between 2^13 and 2^14), so no bf16 query
// overflows or vanishes; an element is rounded only where it is below 2^-24 of its row's largest.
// Weights are rounded to FP16, 2^-12 of each at the most (a product takes both operands in one type, and the scaled codes are
// exact in FP16 with 3 bits to spare; bf16 weights would be 8 times coarser), while their sum is of the FP32 ones.  They are
// 2^(x - ref + 11) with a reference that moves when a score passes it by 4 in the exponent: high in FP16's range, so that a weight
// keeps its 11 bits down to 2^-25 of its row's largest, and what is left out below that is 2^-36 of it at the most.  (A reference
// that moves at 1 would reach 2^-28, but moves so often that verify windows take 158 us instead of 143.  Scales on the weights
// would take fewer instructions, 64 rows of 4,096 81 us, but round the product again, and lose it where a dominant position
// meets small values: no better than 2^-20 of the largest at scales of 2^-3.)  Sums are FP32.
//
// Two ways to cut a launch.  By splits: a 3-D grid of (split of `chunk` positions, heads and query tiles, row), states in the
// workspace as every other decode kernel leaves them: a column's bits do not depend on the launch.  Even
// (CRIT_B200_ATTEND_EVEN): the launch's tiles, rows in order, are dealt out in equal runs to the blocks the device holds at
// once; where a run and a row overlap there is one state, slot = block + row (both only grow along the tiles, so the sum
// names the pair), and merge4_kernel folds a row's consecutive slots.  No block idles while another has two splits to go.
//
// Measured (B200, CUDA events around graphs; HBM's floor at the measured copy bandwidth beside it): 64 rows of 4,096 positions,
// 64 query heads on 8 of 128: 88 us (44), 3.3 TB/s; one row of 200,000, 24 on 4 of 256: 71 us (33); 32 verify windows of 6 columns, 40
// on 8 of 128, FP16: 143 us (27); one row of 777: 11 us, two launches' latency.  Cut into splits of 1,024: 98, 107, 220 and 43 us.
// Bound by instructions at the registers' occupancy: of the 64 rows' launch about 410 a warp and tile (the values' codes 150, the
// keys' 60, scales and softmax the rest) fill 65% of the issue slots with 16 warps an SM, the integer pipe 60%; of the verify
// windows' 710 a tile with 8 warps an SM fill 46%, each warp waiting for its own last result.  The same tiles streamed without the
// products take about 60 us.
#include <mutex>
#include <type_traits>

#include "int4.cuh"
#include "tensor_map.cuh"

namespace crit_b200 {

constexpr int D4_MAX_STAGES = 8;
// Stages between the tile a warp works on and the one its turn refills.  A turn waits until every warp is done with the
// tile whose stage it takes: 3 back instead of 2 the warps may stand further apart (64 rows of 4,096: 87.7 us instead of 90.5, one
// row of 200,000 70.7 instead of 72.2, verify windows 0.7% less).
constexpr int D4_SLACK = 3;
constexpr int D4_MAX_ROWS = 256;              // window rows an even launch lists

// The most kv heads a block takes: the pieces asked of HBM are its heads' bytes of a position (8 against 4: 64 rows of 4,096
// 88 us against 99, verify windows of 6 143 against 147).  The scales of a tile come for every kv head, whatever the block's share:
// 6% of the bytes with 8 of 128 (each read once), 1.18 times the bytes with 32.  The blocks of so many heads an SM is to hold: a warp's accumulators
// decide (the registers of 16 warps are 128 a thread, of 8 warps 255).
constexpr int D4_HEADS = 8;
constexpr __host__ __device__ int decode4_blocks(int d, int nt) { return nt == 1 && d <= 128 ? 2 : 1; }

struct Decode4Launch {
    int heads;              // kv heads a block takes (HB)
    int ctiles;             // tiles of 8 NT query rows a window row takes at most
    int stages;             // of the ring
    int stage_bytes;
    int row;                // bytes of a tensor map's row: 128, or what the block's heads fill of it
    int blocks;             // of an even launch; 0: splits
};

// Two FP16 numbers from the nibbles 0 and 4 (low) or 1 and 5 (high) of a word: n * 2^-24 and 16 n * 2^-24 ...
__device__ __forceinline__ uint32_t raw_low(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t raw_high(uint32_t w) { return w & 0x00f000f0u; }
// ... or n - 8.
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
template <bool RAW>
__device__ __forceinline__ void key_operands(uint32_t lo, uint32_t hi, uint32_t (&a1)[4], uint32_t (&a2)[4]) {
    // words lo and hi -> operands 0 and 1 of the low nibbles, 2 and 3 of the high ones; a2 from the words' upper bytes
    a1[0] = RAW ? raw_low(lo) : codes_low(lo), a1[1] = RAW ? raw_low(hi) : codes_low(hi);
    a1[2] = RAW ? raw_high(lo) : codes_high(lo), a1[3] = RAW ? raw_high(hi) : codes_high(hi);
    lo >>= 8, hi >>= 8;
    a2[0] = RAW ? raw_low(lo) : codes_low(lo), a2[1] = RAW ? raw_low(hi) : codes_low(hi);
    a2[2] = RAW ? raw_high(lo) : codes_high(lo), a2[3] = RAW ? raw_high(hi) : codes_high(hi);
}

__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b) {
    __half2 h = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t hfma2_bits(uint32_t a, uint32_t b, uint32_t c) {
    __half2 h = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), *reinterpret_cast<__half2*>(&c));
    return *reinterpret_cast<uint32_t*>(&h);
}
// The nibbles 1 and 5 of a word as (n - 8) * scale / 128, `scale` a pair over 128 and `less` -72 times that.
__device__ __forceinline__ uint32_t scaled_codes(uint32_t w, uint32_t scale, uint32_t less) { return hfma2_bits((w & 0x00f000f0u) | 0x54005400u, scale, less); }
// D = A * B, and D += A * B (FP16 operands, FP32 sums; not volatile: nothing but the registers is touched, and the compiler
// may place them between the loads and the conversions).
__device__ __forceinline__ void mma16816_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma16816_add(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// all ones in the halves that are not zero
__device__ __forceinline__ uint32_t nonzero2(uint32_t a) { return __hne2_mask(*reinterpret_cast<__half2*>(&a), __floats2half2_rn(0.f, 0.f)); }

__device__ __forceinline__ uint32_t shared_u32(uint32_t at) {
    uint32_t x;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
    return x;
}
__device__ __forceinline__ uint32_t shared_u16(uint32_t at) {
    uint16_t x;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at) : "memory");
    return x;
}
// Lane 0 tells a barrier that the warp is done with a stage (a predicate, no branch).
__device__ __forceinline__ void arrive_lane0(uint32_t bar, int lane) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar), "r"(lane) : "memory");
}

// The scales of two positions for a row's groups, as FP16 pairs (first position, second): NG bytes from each address.
template <int NG>
__device__ __forceinline__ void scale_pairs(uint32_t a, uint32_t b, uint32_t (&pair)[NG]) {
    constexpr int WORDS = NG >= 4 ? NG / 4 : 1;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
        uint32_t x, y;
        if constexpr (NG >= 4) x = shared_u32(a + 4 * w), y = shared_u32(b + 4 * w);
        else x = shared_u16(a), y = shared_u16(b);
#pragma unroll
        for (int k = 0; k < (NG >= 4 ? 2 : 1); ++k) {
            const uint32_t four = __byte_perm(x, y, k ? 0x7632 : 0x5410);          // bytes [x, x', y, y']: two groups
            pair[4 * w + 2 * k] = (four << 7) & 0x7f807f80u;
            pair[4 * w + 2 * k + 1] = (four >> 1) & 0x7f807f80u;
        }
    }
}

// Byte offset of 16-byte chunk c of row `row` of a tile, rows of `bytes` (128, 64 or 32) with TMA's swizzle of that width.
__device__ __forceinline__ uint32_t chunk4(uint32_t row, uint32_t c, uint32_t bytes) {
    const uint32_t turn = bytes == 128 ? row & 7 : (bytes == 64 ? (row >> 1) & 3 : (row >> 2) & 1);
    return row * bytes + ((c ^ turn) << 4);
}

// The positions that a row's page table holds.
__device__ __forceinline__ int64_t table_positions4(const crit_b200_attend_params& p) {
    return p.table_pages > 0 ? (int64_t)p.table_pages * p.page : (int64_t)p.chunk * p.max_splits;
}
// Whether a row begins past its page table: nothing it says can be right.  It is reported; an even launch leaves it out, its
// output as it was, a launch cut into splits reads what the table holds.
__device__ __forceinline__ bool past_table4(const crit_b200_attend_params& p, int r, int count) {
    return count > 0 && p.firsts[r] >= table_positions4(p) + ((p.flags & CRIT_B200_ATTEND_CONTEXT) ? 1 : 0);
}
// A row of the launch: its tiles, as far as its page table goes (a row may end past it where a captured step is padded).
__device__ __forceinline__ int row_tiles4(const crit_b200_attend_params& p, int r, int count) {
    const int64_t end = p.firsts[r] + ((p.flags & CRIT_B200_ATTEND_CONTEXT) ? 0 : count), holds = table_positions4(p), L = end < holds ? end : holds;
    if ((p.flags & CRIT_B200_ATTEND_EVEN) && past_table4(p, r, count)) return 0;
    return count > 0 && L > 0 ? (int)((L + 15) >> 4) : 0;
}
__device__ __forceinline__ int row_count4(const crit_b200_attend_params& p, int r) {
    const int count = p.counts ? p.counts[r] : p.columns;
    return count > p.columns ? p.columns : count;
}

// A place among a block's tiles: row, (head group, query tile) of the row, tile.
struct Place4 {
    int r, sub, tile, tiles, subs;
};

// MASKS: draft trees, sliding windows and block lists (else a column sees every position up to its own).
// FAST: the fewest instructions for the tile's width (the keys' raw codes).  Otherwise every width does the same arithmetic, so
// that a launch cut into splits gives a column the same bits alone and in any window.
template <int D, int NT, bool MASKS, bool FAST>
__global__ void __launch_bounds__(32 * D4_HEADS, decode4_blocks(D, NT))
decode4_kernel(const crit_b200_attend_params p, const Decode4Launch u, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int NG = D / 32;                // groups of a row
    constexpr int ROWS = 8 * NT;
    constexpr int TPI = FAST && NT == 4 ? 1 : 2;        // tiles an iteration takes (the widest has products enough of its own)
    constexpr bool RAW_K = FAST && NT <= 2;                 // the 8 of the keys' codes through the accumulators' start
    // A row's m_run is set TOP below its maximum, so that the largest weight is 2^TOP, and moves when a weight passes 2^SLACK
    // (FAST: with it every row of the tile whose weights passed 2^TOP, so that fewer iterations stop for it).
    constexpr float TOP = 11.f, SLACK = 15.f;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    __shared__ __align__(8) uint64_t bars_mem[2 * D4_MAX_STAGES];
    __shared__ int list_first[D4_MAX_ROWS + 1], list_tiles[D4_MAX_ROWS], list_subs[D4_MAX_ROWS];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int G = p.q_heads / p.kv_heads;
    const int HB = u.heads, HG = p.kv_heads / HB;
    const uint32_t full = smem_addr(bars_mem), empty = full + D4_MAX_STAGES * 8;
    const bool context = (p.flags & CRIT_B200_ATTEND_CONTEXT) != 0;       // the positions before a row's first only
    if (threadIdx.x == 0) {
        for (int s = 0; s < u.stages; ++s) mbar_init(full + s * 8, 1), mbar_init(empty + s * 8, HB);
        mbar_init_fence();
    }

    // -- the block's tiles -------------------------------------------------------------------------------------------------
    Place4 at;                      // where the block begins
    int length;                     // tiles it takes
    if (u.blocks) {
        if (warp == 0) {
            int carry = 0;
            for (int base = 0; base < p.n_rows; base += 32) {
                const int r = base + lane;
                int tiles = 0, subs = 0;
                if (r < p.n_rows) {
                    const int count = row_count4(p, r);
                    tiles = row_tiles4(p, r, count), subs = count > 0 ? HG * ((count * G + ROWS - 1) / ROWS) : 0;
                }
                int scan = tiles * subs;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, scan, o);
                    if (lane >= o) scan += up;
                }
                if (r < p.n_rows) list_first[r + 1] = carry + scan, list_tiles[r] = tiles, list_subs[r] = subs;
                carry += __shfl_sync(0xffffffffu, scan, 31);
            }
            if (lane == 0) list_first[0] = 0;
        }
        __syncthreads();
        const int total = list_first[p.n_rows];
        const int share = (total + u.blocks - 1) / u.blocks, run = share > 1 ? share : 1;
        if (blockIdx.x == 0) {      // what the fold reads: the run, and where a row begins
            int* info = reinterpret_cast<int*>(p.workspace);
            for (int r = threadIdx.x; r <= p.n_rows; r += blockDim.x) info[1 + r] = list_first[r];
            if (threadIdx.x == 0) info[0] = run;
        }
        const int begin = blockIdx.x * run;
        length = total - begin < run ? total - begin : run;
        if (length <= 0) return;
        int lo = 0, hi = p.n_rows;                  // the row whose tiles hold `begin` (of rows that begin there the last, which has tiles)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (list_first[mid] <= begin) lo = mid;
            else hi = mid;
        }
        at.r = lo, at.tiles = list_tiles[lo], at.subs = list_subs[lo];
        at.sub = (begin - list_first[lo]) / at.tiles;
        at.tile = begin - list_first[lo] - at.sub * at.tiles;
    } else {
        __syncthreads();
        const int r = blockIdx.z, count = row_count4(p, r);
        const int hg = blockIdx.y / u.ctiles, ct = blockIdx.y - hg * u.ctiles;
        if (count <= 0 || ct * ROWS >= count * G) return;
        if (blockIdx.x == 0 && threadIdx.x == 0 && p.status && past_table4(p, r, count)) atomicExch(p.status, CRIT_B200_STATUS_PLAN);
        at.r = r, at.tiles = row_tiles4(p, r, count), at.subs = 0x7fffffff;
        at.sub = blockIdx.y, at.tile = blockIdx.x * (p.chunk >> 4);
        length = at.tiles - at.tile < (p.chunk >> 4) ? at.tiles - at.tile : (p.chunk >> 4);
        if (length <= 0) {
            // a row that holds no position (a context row at position 0): zeros and -inf, as the fold of no state gives
            if (at.tiles == 0 && blockIdx.x == 0 && !(p.flags & CRIT_B200_ATTEND_PARTIALS)) {
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
    }

    const int code_bytes = HB * 16 * (D / 2);                              // a tile's keys, or its values
    const int row_scales = p.kv_heads * NG;                                // bytes of a position's scales
    const int scale_bytes = 16 * row_scales;
    const uint32_t tiles_per_page = (uint32_t)p.page >> 4;
    const int tshift = (tiles_per_page & (tiles_per_page - 1)) == 0 ? __ffs((int)tiles_per_page) - 1 : -1;
    const uint32_t pages_total = (uint32_t)(p.slots / p.page);
    const uint32_t ring = smem_addr(smem);

    // -- refilling the ring (lane 0; a warp's turns are HB tiles apart) ------------------------------------------------------
    Place4 next = at;               // the tile of this warp's next turn, its page read ahead
    int next_n = warp, next_page = 0, next_row = 0;
    const int32_t* next_table = nullptr;
    auto step_to = [&](Place4& c, int by) {
        c.tile += by;
        while (c.tile >= c.tiles) {
            c.tile -= c.tiles;
            if (++c.sub >= c.subs) {
                c.sub = 0;
                do ++c.r; while (c.r < p.n_rows && list_tiles[c.r] * list_subs[c.r] == 0);
                if (c.r >= p.n_rows) return;         // (past the launch's last tile: no turn comes to it)
                c.tiles = list_tiles[c.r], c.subs = list_subs[c.r];
            }
        }
    };
    auto read_row = [&]() {         // what stays the same from tile to tile
        next_table = p.tables + (int64_t)p.rows[next.r] * p.table_stride;
        next_row = (u.blocks ? next.sub / (next.subs / HG) : next.sub / u.ctiles) * (HB * (D / 2) / u.row);
    };
    auto read_page = [&]() {
        const uint32_t tile = (uint32_t)next.tile;
        next_page = next_table[tshift >= 0 ? tile >> tshift : tile / tiles_per_page];
    };
    bool outside = false;
    auto refill = [&](int stage) {  // tile next_n into its stage, which is free
        const uint32_t tile = (uint32_t)next.tile;
        outside |= (uint32_t)next_page >= pages_total;             // the tensor's last page is read instead; reported below
        const uint32_t pg = (uint32_t)next_page < pages_total ? (uint32_t)next_page : pages_total - 1;
        const uint32_t slot0 = pg * (uint32_t)p.page + ((tshift >= 0 ? tile & (tiles_per_page - 1) : tile % tiles_per_page) << 4);
        const uint64_t scales0 = (uint64_t)slot0 * (uint32_t)row_scales;
        const uint32_t bar = full + stage * 8, to = ring + stage * u.stage_bytes;
        mbar_expect_tx(bar, (uint32_t)(2 * code_bytes + 2 * scale_bytes));
        tma_load_3d(to, &kmap, 0, (int)slot0, next_row, bar);
        bulk_load(to + 2 * code_bytes, (const char*)p.key_scales + scales0, scale_bytes, bar);
        tma_load_3d(to + code_bytes, &vmap, 0, (int)slot0, next_row, bar);
        bulk_load(to + 2 * code_bytes + scale_bytes, (const char*)p.value_scales + scales0, scale_bytes, bar);
    };
    auto turn_over = [&]() {        // to this warp's next turn
        next_n += HB;
        if (lane == 0 && next_n < length) {
            next.tile += HB;
            if (next.tile >= next.tiles) step_to(next, 0), read_row();
            read_page();
        }
    };
    if (lane == 0 && warp < length) step_to(next, warp), read_row(), read_page();
    while (next_n < u.stages - D4_SLACK && next_n < length) {      // the first tiles: D4_SLACK stages stay free
        if (lane == 0) refill(next_n);
        turn_over();
    }

    bool dead = false;
    int n = 0, stage = 0;           // tiles taken, the ring's place
    uint32_t phase = 0;
    // ldmatrix rows: lanes 0-7 and 8-15 name positions 0-7 and 8-15 of the head's chunk 2 i, lanes 16-31 the same of chunk 2 i + 1
    // (whose address is that of chunk 0 or 1 with the bits of 2 i changed: a head's chunks begin at a multiple of their number)
    const uint32_t heads_row = (uint32_t)u.row / (D / 2);
    const uint32_t lane_codes = ring + chunk4(warp / heads_row * 16 + (lane & 7) + 8 * ((lane >> 3) & 1), warp % heads_row * NG + (lane >> 4), u.row);

    while (n < length) {
        // -- a unit: the tiles of one row, head group and query tile in this block -----------------------------------------
        const int r = at.r, count = row_count4(p, r);
        const int64_t holds = table_positions4(p), first = p.firsts[r] < holds ? p.firsts[r] : holds;
        const int first32 = (int)first;
        const int per_hg = u.blocks ? at.subs / HG : u.ctiles;
        const int hg = at.sub / per_hg, ct = at.sub - hg * per_hg;
        const int h = hg * HB + warp, start = p.starts[r];
        const uint32_t lane_kscales = ring + 2 * code_bytes + h * NG + g * row_scales;
        const uint32_t lane_vscales = ring + 2 * code_bytes + scale_bytes + h * NG + 2 * t * row_scales;
        const int tile0 = at.tile, ntiles = at.tiles - tile0 < length - n ? at.tiles - tile0 : length - n;

        uint32_t qb[NT][NG][4];                    // pairs (0, 4), (1, 5), (2, 6), (3, 7) of elements 32 group + 8 t + ..
        uint32_t q8[RAW_K ? NT : 1][2];            // -8 * the sums of the groups' queries as an operand: two FP16 terms of groups 2 t, 2 t + 1
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
            const bool bf16 = p.q_dtype == CRIT_B200_DTYPE_BF16;
            auto element = [&](int k, int i) {
                const uint32_t w = (&raw[k].x)[i >> 1];
                if (bf16) return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
                return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w >> 16 : w)));
            };
            {   // the largest magnitude: both types' bits without the sign are in the order of their values
                uint32_t high = 0u;
#pragma unroll
                for (int k = 0; k < NG; ++k)
                    high = __vmaxu2(high, __vmaxu2(__vmaxu2(raw[k].x & 0x7fff7fffu, raw[k].y & 0x7fff7fffu), __vmaxu2(raw[k].z & 0x7fff7fffu, raw[k].w & 0x7fff7fffu)));
                high = max(high >> 16, high & 0xffffu);
                amax = bf16 ? __uint_as_float(high << 16) : __half2float(__ushort_as_half((unsigned short)high));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            int e = (int)((__float_as_uint(amax) >> 23) & 255u) - 127 - 13;
            e = amax > 0.f ? (e < -90 ? -90 : (e > 90 ? 90 : e)) : 0;
            const float down = __int_as_float(((127 - e) << 23) | (p.scale < 0.f ? (int)0x80000000 : 0));       // (mul is not negative)
            if constexpr (RAW_K) q8[nt][0] = q8[nt][1] = 0u;
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float part = RAW_K && (j & 1) ? 0.0625f : 1.f;            // (the odd nibbles' operands are 16 n)
                    qb[nt][k][j] = pack2<false>(element(k, j) * down * part, element(k, j + 4) * down * part);
                    const float2 back = __half22float2(*reinterpret_cast<__half2*>(&qb[nt][k][j]));
                    sum += (back.x + back.y) * (RAW_K && (j & 1) ? 16.f : 1.f);
                }
                if constexpr (RAW_K) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    sum *= -0x1p-21f;                                                  // (8 * 2^-24)
                    const __half hi = __float2half_rn(sum), lo = __float2half_rn(sum - __half2float(hi));
                    if (2 * t == (k & ~1)) {
                        q8[nt][0] |= (uint32_t)__half_as_ushort(hi) << (16 * (k & 1));
                        q8[nt][1] |= (uint32_t)__half_as_ushort(lo) << (16 * (k & 1));
                    }
                }
            }
            // the lane's columns are query rows 2 t and 2 t + 1: their exponents live with lanes g = 2 t and 2 t + 1
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int er = __shfl_sync(0xffffffffu, e, (2 * t + j) * 4);
                mul[nt][j] = fmaxf(fabsf(p.scale) * LOG2E * __int_as_float((127 + er + (RAW_K ? 24 : 0)) << 23), 1e-37f);
                const int c = (ct * ROWS + nt * 8 + 2 * t + j) / G;
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

        // An iteration over `have` tiles from tile i of the unit.  GENERAL false: TPI tiles that every query row sees whole, the
        // bulk of a long row, in code of its own so that no instruction of it is about masks.
        auto iterate = [&](auto general, const int i, const int have) {
            constexpr bool GENERAL = decltype(general)::value;
            float x[TPI][NT][4];
            int stages[TPI];
#pragma unroll
            for (int v = 0; v < TPI; ++v) {
                if (GENERAL && v >= have) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) x[v][nt][c] = -INFINITY;
                    continue;
                }
                // this warp's turn: tile n + S - 3 into the stage of tile n - 3, once every warp is done with that
                if (n + u.stages - D4_SLACK == next_n) {
                    if (lane == 0 && next_n < length) {
                        int to = stage - D4_SLACK;
                        to = to < 0 ? to + u.stages : to;
                        // the stage's uses so far are (n - 3) / S whole rounds and one: wait for the end of the last
                        if (n < D4_SLACK || mbar_wait(empty + to * 8, (uint32_t)((n - D4_SLACK) / u.stages) & 1u)) refill(to);
                        else dead = true;
                    }
                    turn_over();
                }
                stages[v] = stage;
                if (!mbar_wait(full + stage * 8, phase)) dead = true;
                __syncwarp();
                if (++stage == u.stages) stage = 0, phase ^= 1;
                ++n;
                // scores
                const uint32_t from = stages[v] * u.stage_bytes;
                uint32_t pair[NG];
                scale_pairs<NG>(lane_kscales + from, lane_kscales + from + 8 * row_scales, pair);
                if constexpr (RAW_K) {
                    // scale[position][group] * (-8 * sum of the group's queries): groups 2 t and 2 t + 1 are this lane's columns
                    uint32_t even = pair[0], odd = pair[1];
#pragma unroll
                    for (int k = 2; k < NG; k += 2) even = 2 * t == k ? pair[k] : even, odd = 2 * t == k ? pair[k + 1] : odd;
                    uint32_t a[4];
                    a[0] = a[2] = __byte_perm(even, odd, 0x5410), a[1] = a[3] = __byte_perm(even, odd, 0x7632);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816_new(x[v][nt], a, q8[nt][0], q8[nt][1]);
                }
#pragma unroll
                for (int k = 0; k < NG; k += 2) {
                    uint32_t w[4];
                    ldmatrix_x4(w, (lane_codes + from) ^ (k << 4));
#pragma unroll
                    for (int o = 0; o < 2; ++o) {
                        const float2 s = __half22float2(*reinterpret_cast<__half2*>(&pair[k + o]));
                        uint32_t a1[4], a2[4];
                        key_operands<RAW_K>(w[2 * o], w[2 * o + 1], a1, a2);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float c[4];
                            mma16816_new(c, a1, qb[nt][k + o][0], qb[nt][k + o][1]);
                            mma16816_add(c, a2, qb[nt][k + o][2], qb[nt][k + o][3]);
                            if (!RAW_K && k + o == 0) {
                                x[v][nt][0] = c[0] * s.x, x[v][nt][1] = c[1] * s.x, x[v][nt][2] = c[2] * s.y, x[v][nt][3] = c[3] * s.y;
                            } else {
                                x[v][nt][0] = fmaf(c[0], s.x, x[v][nt][0]), x[v][nt][1] = fmaf(c[1], s.x, x[v][nt][1]);
                                x[v][nt][2] = fmaf(c[2], s.y, x[v][nt][2]), x[v][nt][3] = fmaf(c[3], s.y, x[v][nt][3]);
                            }
                        }
                    }
                }
            }

            // masks, online softmax
            bool passed = false;
            float top[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int v = 0; v < TPI; ++v)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float y = x[v][nt][c];
                        if constexpr (GENERAL) {
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
                top[nt][0] = mx[0] * mul[nt][0], top[nt][1] = mx[1] * mul[nt][1];
                passed |= top[nt][0] > m_run[nt][0] + SLACK || top[nt][1] > m_run[nt][1] + SLACK;
            }
            // The reference of a row moves only when a score passes it; the lanes' maxima are compared across the warp, and the
            // sums brought to the new reference, only then.
            if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float alpha[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float high = top[nt][j];
                        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 4));
                        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 8));
                        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 16));
                        const bool moved = high > m_run[nt][j] + (FAST ? TOP : SLACK);
                        alpha[j] = moved ? ex2(m_run[nt][j] - (high - TOP)) : 1.f;
                        m_run[nt][j] = moved ? high - TOP : m_run[nt][j];
                        l_run[nt][j] *= alpha[j];
                    }
#pragma unroll
                    for (int k = 0; k < NG; ++k)
#pragma unroll
                        for (int c = 0; c < 8; ++c) acc[k][c >> 2][nt][c & 3] *= alpha[c & 1];
                }
            }
            uint32_t pb[TPI][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                // (a row that has seen nothing has no reference: its scores are all -inf)
                const float sub[2] = {GENERAL && m_run[nt][0] == -INFINITY ? 0.f : m_run[nt][0], GENERAL && m_run[nt][1] == -INFINITY ? 0.f : m_run[nt][1]};
#pragma unroll
                for (int v = 0; v < TPI; ++v) {
                    float w[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        w[c] = ex2(fmaf(x[v][nt][c], mul[nt][c & 1], -sub[c & 1]));
                        l_run[nt][c & 1] += w[c];
                    }
                    pb[v][nt][0] = transposed8(pack2<false>(w[0], w[1]));
                    pb[v][nt][1] = transposed8(pack2<false>(w[2], w[3]));
                }
            }

            // outputs
#pragma unroll
            for (int v = 0; v < TPI; ++v) {
                if (GENERAL && v >= have) continue;
                const uint32_t from = stages[v] * u.stage_bytes;
                uint32_t pair[2][NG];                    // scales of positions 2 t, 2 t + 1 and of 2 t + 8, 2 t + 9
                scale_pairs<NG>(lane_vscales + from, lane_vscales + from + row_scales, pair[0]);
                scale_pairs<NG>(lane_vscales + from + 8 * row_scales, lane_vscales + from + 9 * row_scales, pair[1]);
                if constexpr (GENERAL) {
                    // A position that a query row does not take may have any scale, a NaN too: the scale becomes 0, and the
                    // weights of the rows that do take the position a NaN.
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        uint32_t bad = 0u;
#pragma unroll
                        for (int k = 0; k < NG; ++k) {
                            const uint32_t odd = __vcmpgeu2(pair[hf][k], 0x7c007c00u);
                            pair[hf][k] &= ~odd, bad |= odd;
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) pb[v][nt][hf] |= nonzero2(pb[v][nt][hf]) & bad;
                    }
                }
#pragma unroll
                for (int k = 0; k < NG; k += 2) {
                    uint32_t w[4];
                    ldmatrix_x4_trans(w, (lane_codes + from + code_bytes) ^ (k << 4));
#pragma unroll
                    for (int o = 0; o < 2; ++o) {
                        // words of positions 0-7 and 8-15: values 4 g .. 4 g + 3 of the group
                        const uint32_t s0 = hmul2_bits(pair[0][k + o], 0x20002000u), s1 = hmul2_bits(pair[1][k + o], 0x20002000u);        // / 128
                        const uint32_t c0 = hmul2_bits(pair[0][k + o], 0xb880b880u), c1 = hmul2_bits(pair[1][k + o], 0xb880b880u);        // * -72 / 128
                        const uint32_t lo = w[2 * o], hi = w[2 * o + 1];
                        const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
                        const uint32_t a1[4] = {hmul2_bits(codes_low(lo), s0), scaled_codes(lo, s0, c0), hmul2_bits(codes_low(hi), s1), scaled_codes(hi, s1, c1)};
                        const uint32_t a2[4] = {hmul2_bits(codes_low(lo8), s0), scaled_codes(lo8, s0, c0), hmul2_bits(codes_low(hi8), s1), scaled_codes(hi8, s1, c1)};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816_add(acc[k + o][0][nt], a1, pb[v][nt][0], pb[v][nt][1]);
                            mma16816_add(acc[k + o][1][nt], a2, pb[v][nt][0], pb[v][nt][1]);
                        }
                    }
                }
                __syncwarp();
                arrive_lane0(empty + stages[v] * 8, lane);
            }
        };
        // (a wait that ran out ends the warp's work after its iteration; what it computed is not written)
        int i = 0;
        if constexpr (!MASKS) {
            const int clear = (first32 >> 4) - tile0;           // tiles whose positions are all before the row's first
            const int plain = (clear < ntiles ? clear : ntiles) / TPI * TPI;
            for (; i < plain && !__any_sync(0xffffffffu, dead); i += TPI) iterate(std::false_type(), i, TPI);
        }
        for (; i < ntiles && !__any_sync(0xffffffffu, dead); i += TPI) iterate(std::true_type(), i, ntiles - i < TPI ? ntiles - i : TPI);
        if (__any_sync(0xffffffffu, dead)) break;

        // -- the state, or the row's output ------------------------------------------------------------------------------------
        bool whole, fits = true;
        int64_t state0 = 0, states = 0;                         // an even launch: rows of states before this one's, their number
        int prow0 = 0, split = 0;
        if (u.blocks) {
            whole = ntiles == at.tiles && !p.sinks;
            states = ((int64_t)u.blocks + (int64_t)p.n_rows * HG * u.ctiles) * HB * ROWS;
            state0 = ((int64_t)blockIdx.x + ((int64_t)r * HG + hg) * u.ctiles + ct) * HB * ROWS + warp * ROWS;
        } else {
            split = blockIdx.x;
            whole = at.tiles <= (p.chunk >> 4) && !(p.flags & CRIT_B200_ATTEND_PARTIALS) && !p.sinks;     // (sinks join in the fold)
            states = (int64_t)p.partial_rows * p.q_heads * p.max_splits;
            prow0 = p.offsets ? p.offsets[r] - p.offsets[0] : r * p.columns;
            fits = whole || (p.workspace && split < p.max_splits && prow0 >= 0 && prow0 + count <= p.partial_rows);
            if (!fits && lane == 0 && p.status) atomicExch(p.status, CRIT_B200_STATUS_PLAN);
        }
        float* const space = p.workspace + (u.blocks ? (p.n_rows + 2 + 31) / 32 * 32 : 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float l = l_run[nt][j];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                const int row = nt * 8 + 2 * t + j, flat = ct * ROWS + row;
                const int col = flat / G, gq = flat - col * G;
                if (col >= count || !fits) continue;
                const int token = start + col, head = h * G + gq;
                const float inv = whole ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;          // (a NaN stays one)
                auto value = [&](int k, int e) {                 // element 32 k + 4 g + e
                    return acc[k][e >> 1][nt][(e & 1) * 2 + j] * (128.f * inv);
                };
                if (whole) {
                    char* dst = (char*)p.out + ((int64_t)token * p.out_stride_token + (int64_t)head * p.out_stride_head + 4 * g) * 2;
#pragma unroll
                    for (int k = 0; k < NG; ++k)
                        *reinterpret_cast<uint2*>(dst + k * 64) = p.q_dtype == CRIT_B200_DTYPE_BF16
                                                                      ? make_uint2(pack2<true>(value(k, 0), value(k, 1)), pack2<true>(value(k, 2), value(k, 3)))
                                                                      : make_uint2(pack2<false>(value(k, 0), value(k, 1)), pack2<false>(value(k, 2), value(k, 3)));
                    if (p.lse && g == 0) p.lse[(int64_t)token * p.q_heads + head] = l == 0.f ? -INFINITY : m_run[nt][j] * LN2 + logf(l);
                } else {
                    const int64_t where = u.blocks ? state0 + row : ((int64_t)(prow0 + col) * p.q_heads + head) * p.max_splits + split;
                    float* dst = space + where * D + 4 * g;
#pragma unroll
                    for (int k = 0; k < NG; ++k) *reinterpret_cast<float4*>(dst + k * 32) = make_float4(value(k, 0), value(k, 1), value(k, 2), value(k, 3));
                    if (g == 0) {
                        space[states * D + where] = m_run[nt][j];
                        space[states * (D + 1) + where] = l;
                    }
                }
            }
        step_to(at, ntiles);
    }
    if (outside && p.status) atomicExch(p.status, CRIT_B200_STATUS_BOUNDS);
    if (__syncthreads_or(dead ? 1 : 0) && threadIdx.x == 0) {
        // a copy or a reader never came: the copies in flight get a last bounded chance to land
        for (int s = 0; s < u.stages; ++s) mbar_wait(full + s * 8, 0, 1000000ull), mbar_wait(full + s * 8, 1, 1000000ull);
        if (p.status) atomicExch(p.status, CRIT_B200_STATUS_TMA);
    }
}

// The fold of an even launch: a row's states are consecutive slots.  WARPS warps serve a (window token, query head), warp w the
// slots w, w + WARPS, ..; the warps' sums are added in warp order.
template <int D, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) merge4_kernel(const crit_b200_attend_params p, const Decode4Launch u, const int rows_tile) {
    constexpr int PER = D / 32;
    __shared__ __align__(8) float part_m[WARPS], part_l[WARPS], part_o[WARPS > 1 ? WARPS : 1][WARPS > 1 ? D : 1];
    const int lane = threadIdx.x & 31, warp = WARPS == 1 ? 0 : threadIdx.x >> 5;
    const int head = WARPS == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x, col = blockIdx.y, r = blockIdx.z;
    if (head >= p.q_heads) return;
    const int* info = reinterpret_cast<const int*>(p.workspace);
    const int run = info[0], first = info[1 + r];
    const int count = row_count4(p, r), start = p.starts[r];
    const int tiles = row_tiles4(p, r, count);
    if (col >= count) return;
    if (past_table4(p, r, count)) {
        if (lane == 0 && p.status) atomicExch(p.status, CRIT_B200_STATUS_PLAN);
        return;
    }
    const int G = p.q_heads / p.kv_heads, HB = u.heads, HG = p.kv_heads / HB;
    const int h = head / G, hg = h / HB, flat = col * G + head - h * G, ct = flat / rows_tile;
    const int ctiles = (count * G + rows_tile - 1) / rows_tile;
    int lo = 0, n = 0;
    if (tiles > 0) {
        const int begin = first + (hg * ctiles + ct) * tiles;
        lo = begin / run, n = (begin + tiles - 1) / run - lo + 1;
        if (n == 1 && !p.sinks) return;                              // written by the first launch
    }
    const float* space = p.workspace + (p.n_rows + 2 + 31) / 32 * 32;
    const int64_t slots = (int64_t)u.blocks + (int64_t)p.n_rows * HG * u.ctiles;
    const int per = HB * rows_tile;
    const int64_t state0 = ((int64_t)lo + ((int64_t)r * HG + hg) * u.ctiles + ct) * per + (h - hg * HB) * rows_tile + (flat - ct * rows_tile);
    const float* pm = space + slots * per * D + state0;
    const float* pl = pm + slots * per;
    const float* po = space + state0 * D + lane * PER;
    // a warp's states four at a time, everything of them asked for at once; the maximum and the sums go along
    float top = -INFINITY, total = 0.f, acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
    for (int s0 = warp; s0 < n; s0 += 4 * WARPS) {
        float m[4], l[4], v[4][PER];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int s = s0 + k * WARPS;
            m[k] = -INFINITY, l[k] = 0.f;
#pragma unroll
            for (int i = 0; i < PER; ++i) v[k][i] = 0.f;
            if (s >= n) continue;
            m[k] = pm[(int64_t)s * per], l[k] = pl[(int64_t)s * per];
            const float* o = po + (int64_t)s * per * D;
            if constexpr (PER == 2) {
                const float2 a = *reinterpret_cast<const float2*>(o);
                v[k][0] = a.x, v[k][1] = a.y;
            } else {
#pragma unroll
                for (int i = 0; i < PER; i += 4) {
                    const float4 a = *reinterpret_cast<const float4*>(o + i);
                    v[k][i] = a.x, v[k][i + 1] = a.y, v[k][i + 2] = a.z, v[k][i + 3] = a.w;
                }
            }
        }
        const float up = fmaxf(fmaxf(top, fmaxf(m[0], m[1])), fmaxf(m[2], m[3])), sub = up == -INFINITY ? 0.f : up;
        const float keep = ex2(top - sub);
        total *= keep;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] *= keep;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float w = ex2(m[k] - sub);
            total = fmaf(l[k], w, total);
#pragma unroll
            for (int i = 0; i < PER; ++i) acc[i] = fmaf(v[k][i], w, acc[i]);
        }
        top = up;
    }
    if constexpr (WARPS > 1) {
        if (lane == 0) part_m[warp] = top, part_l[warp] = total;
#pragma unroll
        for (int i = 0; i < PER; ++i) part_o[warp][lane * PER + i] = acc[i];
        __syncthreads();
        if (threadIdx.x >= D / 2) return;                  // two columns a thread
        top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, part_m[w]);
        const float sub = top == -INFINITY ? 0.f : top;
        total = acc[0] = acc[1] = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = ex2(part_m[w] - sub);
            const float2 o = *reinterpret_cast<const float2*>(&part_o[w][2 * threadIdx.x]);
            total = fmaf(part_l[w], f, total), acc[0] = fmaf(o.x, f, acc[0]), acc[1] = fmaf(o.y, f, acc[1]);
        }
    }
    constexpr int MINE = WARPS > 1 ? 2 : PER;               // columns this thread writes, from `at`
    const int at = WARPS > 1 ? 2 * threadIdx.x : lane * PER;
    float shrink = 1.f;                     // the head's sink, last: one position more without a value
    if (p.sinks) sink_fold(p.sinks[head], top, total, shrink);
    const float inv = total > 0.f ? shrink / total : (total == 0.f ? 0.f : total);         // (a NaN stays one)
    const int64_t to = (int64_t)(start + col) * p.out_stride_token + (int64_t)head * p.out_stride_head + at;
#pragma unroll
    for (int i = 0; i < MINE; i += 2)
        *reinterpret_cast<uint32_t*>((char*)p.out + (to + i) * 2) =
            p.q_dtype == CRIT_B200_DTYPE_BF16 ? pack2<true>(acc[i] * inv, acc[i + 1] * inv) : pack2<false>(acc[i] * inv, acc[i + 1] * inv);
    if (p.lse && at == 0) p.lse[(int64_t)(start + col) * p.q_heads + head] = total == 0.f ? -INFINITY : top * LN2 + logf(total);
}

// -- host side --------------------------------------------------------------------------------------------------------------
typedef void (*decode4_fn)(const crit_b200_attend_params, const Decode4Launch, const CUtensorMap, const CUtensorMap);

template <int D, int NT>
static decode4_fn decode4_of(bool masks, bool fast) {
    if (fast) return masks ? decode4_kernel<D, NT, true, true> : decode4_kernel<D, NT, false, true>;
    return masks ? decode4_kernel<D, NT, true, false> : decode4_kernel<D, NT, false, false>;
}

static decode4_fn decode4_pick(int d, int nt, bool masks, bool fast) {
    switch (d) {
        case 64: return nt == 1 ? decode4_of<64, 1>(masks, fast) : (nt == 2 ? decode4_of<64, 2>(masks, fast) : decode4_of<64, 4>(masks, fast));
        case 128: return nt == 1 ? decode4_of<128, 1>(masks, fast) : (nt == 2 ? decode4_of<128, 2>(masks, fast) : decode4_of<128, 4>(masks, fast));
        case 256: return nt == 1 ? decode4_of<256, 1>(masks, fast) : decode4_of<256, 2>(masks, fast);
        default: return nullptr;
    }
}

struct Decode4Plan {
    decode4_fn fn;
    Decode4Launch u;
    int nt, smem, sms, per_sm;
};

// Blocks of a kernel an SM of the current device holds, remembered per kernel, block, shared memory and device.
static int resident4(const void* fn, int threads, int smem, int* sms) {
    struct Entry { const void* fn; int threads, smem, device, per_sm, sms; };
    static Entry seen[256];
    static int n = 0;
    static std::mutex guard;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return 0;
    std::lock_guard<std::mutex> lock(guard);
    for (int i = 0; i < n; ++i)
        if (seen[i].fn == fn && seen[i].threads == threads && seen[i].smem == smem && seen[i].device == device) {
            *sms = seen[i].sms;
            return seen[i].per_sm;
        }
    int per_sm = 0;
    if (cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
        cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, threads, smem) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (n < 256) seen[n++] = Entry{fn, threads, smem, device, per_sm, *sms};
    return per_sm;
}

// The launch of a geometry: kernel, heads a block takes, stages that the blocks' shares of an SM hold, blocks of an even launch.
static int plan4(int q_heads, int kv_heads, int d, int columns, int n_rows, bool masks, bool even, Decode4Plan* out) {
    if (d != 64 && d != 128 && d != 256) return CRIT_B200_EUNSUPPORTED;
    const int rows = columns * (q_heads / kv_heads);
    const int nt = rows <= 8 ? 1 : (rows <= 16 || d == 256 ? 2 : 4);
    Decode4Launch& u = out->u;
    u.heads = D4_HEADS;
    while (kv_heads % u.heads) u.heads >>= 1;
    u.ctiles = (rows + 8 * nt - 1) / (8 * nt);
    u.row = u.heads * d / 2 < 128 ? u.heads * d / 2 : 128;
    u.stage_bytes = (u.heads * 16 * d + 2 * 16 * kv_heads * (d / 32) + 1023) / 1024 * 1024;
    const int blocks = decode4_blocks(d, nt) * D4_HEADS / u.heads;           // (the registers hold as many)
    const int room = (228 * 1024) / blocks - 1024 - 1024 - 4096;                          // (alignment, the driver's, the row lists)
    const int stages = room / u.stage_bytes;
    u.stages = stages < 4 ? 4 : (stages > D4_MAX_STAGES ? D4_MAX_STAGES : stages);
    out->nt = nt, out->smem = 1024 + u.stages * u.stage_bytes;
    if (out->smem > 220 * 1024) return CRIT_B200_EUNSUPPORTED;
    out->fn = decode4_pick(d, nt, masks, even);
    u.blocks = 0, out->sms = out->per_sm = 0;
    if (even) {
        out->per_sm = resident4((const void*)out->fn, 32 * u.heads, out->smem, &out->sms);
        if (out->per_sm < 1 || n_rows > D4_MAX_ROWS) return CRIT_B200_EUNSUPPORTED;
        u.blocks = out->sms * out->per_sm;
    }
    return 0;
}

static int plan4(const crit_b200_attend_params& p, Decode4Plan* out) {
    const bool even = (p.flags & CRIT_B200_ATTEND_EVEN) != 0;
    if (even && (p.flags & CRIT_B200_ATTEND_PARTIALS)) return CRIT_B200_EUNSUPPORTED;
    return plan4(p.q_heads, p.kv_heads, p.head_dim, p.columns, p.n_rows, p.parents || p.sliding > 0 || p.blocks, even, out);
}

// Floats of an even launch's workspace: where the rows begin, and (dim + 2) a state row.
int64_t even_floats4(const crit_b200_attend_params& p) {
    Decode4Plan plan;
    if (p.kind != CRIT_B200_KIND_INT4 || p.head_dim != p.value_dim) return CRIT_B200_EUNSUPPORTED;
    if (int e = plan4(p, &plan)) return e;
    // (the launch's tiles are counted in 32 bits)
    const int64_t holds = p.table_pages > 0 ? (int64_t)p.table_pages * p.page : (int64_t)p.chunk * p.max_splits;
    if (holds > 0x7fffffffLL || (holds / 16 + 1) * p.n_rows > 0x7fffffffLL / ((int64_t)p.kv_heads / plan.u.heads * plan.u.ctiles)) return CRIT_B200_EUNSUPPORTED;
    const int64_t slots = (int64_t)plan.u.blocks + (int64_t)p.n_rows * (p.kv_heads / plan.u.heads) * plan.u.ctiles;
    return (p.n_rows + 2 + 31) / 32 * 32 + slots * plan.u.heads * 8 * plan.nt * (p.head_dim + 2);
}

int launch_decode4(const crit_b200_attend_params& p, cudaStream_t s) {
    if (p.flags & (CRIT_B200_ATTEND_TCGEN05 | CRIT_B200_ATTEND_TCGEN05P | CRIT_B200_ATTEND_TCGEN05T)) return CRIT_B200_EUNSUPPORTED;
    if (p.head_dim != p.value_dim || p.slots < 16 || p.slots > 0x7fffffffLL || p.slots < p.page) return CRIT_B200_EUNSUPPORTED;
    if (!aligned(p.key_scales, 16) || !aligned(p.value_scales, 16)) return CRIT_B200_EALIGN;
    // (positions are 32 bits in the kernel; splits wholly past the table would leave no state for the fold)
    if (p.table_pages < 0 || (int64_t)p.table_pages * p.page > 0x7fffffffLL) return CRIT_B200_EUNSUPPORTED;
    if (!(p.flags & CRIT_B200_ATTEND_EVEN) && p.table_pages > 0 && (int64_t)p.chunk * (p.max_splits - 1) >= (int64_t)p.table_pages * p.page) return CRIT_B200_EINVAL;
    Decode4Plan plan;
    if (int e = plan4(p, &plan)) return e;
    const Decode4Launch& u = plan.u;
    CUtensorMap kmap, vmap;
    if (!rows4_map(&kmap, p.key_pages, p.head_dim, p.kv_heads, u.heads, u.row, p.slots) ||
        !rows4_map(&vmap, p.value_pages, p.head_dim, p.kv_heads, u.heads, u.row, p.slots))
        return CRIT_B200_EUNSUPPORTED;
    cudaError_t ce = cudaFuncSetAttribute((const void*)plan.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, plan.smem);
    if (ce != cudaSuccess) return (int)ce;
    const int64_t hg = p.kv_heads / u.heads;
    if (hg * u.ctiles > 65535 || p.n_rows > 65535) return CRIT_B200_EUNSUPPORTED;
    const dim3 grid = u.blocks ? dim3((unsigned)u.blocks) : dim3((unsigned)p.max_splits, (unsigned)(hg * u.ctiles), (unsigned)p.n_rows);
    plan.fn<<<grid, 32 * u.heads, plan.smem, s>>>(p, u, kmap, vmap);
    CRIT_CHECK_LAUNCH();
    return 0;
}

template <int D>
static void launch_merge4_of(const crit_b200_attend_params& p, const Decode4Plan& plan, bool many, cudaStream_t s) {
    const unsigned heads = (unsigned)p.q_heads, columns = (unsigned)p.columns, rows = (unsigned)p.n_rows;        // (rows <= D4_MAX_ROWS)
    if (many) merge4_kernel<D, 16><<<dim3(heads, columns, rows), 512, 0, s>>>(p, plan.u, 8 * plan.nt);
    else merge4_kernel<D, 1><<<dim3((heads + 3) / 4, columns, rows), 128, 0, s>>>(p, plan.u, 8 * plan.nt);
}

int launch_merge4(const crit_b200_attend_params& p, cudaStream_t s) {
    Decode4Plan plan;
    if (int e = plan4(p, &plan)) return e;
    // Few rows share the blocks: a row may have a state in each, so 16 warps fold it; many rows have a few states each, a warp's
    // work.  One row of 200,000: 71 us, with a warp 164; 64 rows of 4,096: 88 us, with 16 warps 123 (launch and fold together).
    const bool many = (int64_t)p.n_rows * (p.kv_heads / plan.u.heads) * plan.u.ctiles * 16 < plan.u.blocks;
    switch (p.head_dim) {
        case 64: launch_merge4_of<64>(p, plan, many, s); break;
        case 128: launch_merge4_of<128>(p, plan, many, s); break;
        case 256: launch_merge4_of<256>(p, plan, many, s); break;
        default: return CRIT_B200_EUNSUPPORTED;
    }
    CRIT_CHECK_LAUNCH();
    return 0;
}

int plan_decode4(int q_heads, int kv_heads, int d, int columns, int32_t* out5) {
    Decode4Plan plan;
    if (int e = plan4(q_heads, kv_heads, d, columns, 1, false, false, &plan)) return e;
    int sms = 0;
    const int per_sm = resident4((const void*)plan.fn, 32 * plan.u.heads, plan.smem, &sms);
    out5[0] = 1024, out5[1] = plan.smem, out5[2] = 8 * plan.nt, out5[3] = per_sm, out5[4] = sms;
    return 0;
}

}  // namespace crit_b200
