// Matrix products of vocab_ce.hip: C[m, n] = sum_k A[m, k] B[n, k] on v_mfma_f32_32x32x16_f16.
//
// Every matrix lies in memory as PANELS: 32 columns of all rows, 64 bytes per row, row after row; panel after panel.  A tile of rows
// is then one contiguous piece per panel, whichever way it is used: with the columns as k ("KC", one panel per step) or with the
// rows as k ("KS", 32 rows of several panels per step; the transposing LDS read hands the matrix core its layout, so no transposed
// copy of anything is ever made).  Row-major rows of 64 bytes per step were half cache lines: 4.0e8 instead of 2.0e8 L2 requests for
// 16384 x 65536 x 1024.  Row counts are multiples of 256, so nothing is clamped.
//
// SPLIT matrices carry fp32 values as two fp16 numbers, x = hi + lo (22 bits; what is left is below 2^-22 of x); a panel is 16 columns,
// a row of it 16 hi | 16 lo.  A product is hi*hi + hi*lo + lo*hi, three matrix instructions into one fp32 accumulator: 2500 / 3
// TFLOP/s of matrix rate where v_mfma_f32_* has 157.
//
// A step (32 k values, 16 split ones: 64 bytes per tile row) is staged by global_load_lds into a ring of LDS buffers, several steps
// ahead of the one that is multiplied; one barrier per step.  global_load_lds writes linearly, so bank swizzles are applied to the
// global address: KC rows put chunk c (16 bytes) at c ^ ((row >> 2) & 3): sixteen consecutive rows cover all 64 banks.  The four k rows
// of a transposing read are 256 contiguous bytes as they are; split ones take 32 of every 64 bytes from two panels, so odd panels
// change their halves.
#pragma once
#include "vocab_types.h"

#include <type_traits>

namespace tnp {

typedef half_t half8 __attribute__((ext_vector_type(8)));
typedef int int2v __attribute__((ext_vector_type(2)));
typedef int int4v __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

#define TNP_LDS __attribute__((address_space(3)))
#define TNP_GLB __attribute__((address_space(1)))

// Rows of an operand that is read as KS (its rows are the k of the product) may lie in memory on scales of their own, row r by `shift`
// binades (<= 0) below the top one's.  Rows are taken by CLASSES of sixteen binades, one run of the product each, from the smallest numbers to
// the largest: a run multiplies the operand, in registers, by 2^(shift + 16 class) where the row is of its class and by zero elsewhere,
// and the accumulator is brought onto the next class's scale in between.  No row's bits are lost to another's size, and an
// operand whose rows share one scale (class 0 alone, no shifts) needs none of it.  A run goes from the first to the last step that has a row of
// its class, so that a few such rows cost little.
//
// A row's scale is one word: class << 16 | that fp16 number.  A wave reads a step's words by scalar loads (vector loads would wait for the tiles in
// flight), one step ahead: forward and backward of 24576 x 1024 x 128 fp32 with one row 2^40 times as large 232 us (vector loads 488), without such a
// row 148; a run with scales takes 1.4 times one without.
static constexpr int ROW_CLASSES = 32;
__device__ __forceinline__ int row_class(int shift) {
    const int c = -shift >> 4;
    return c < ROW_CLASSES ? c : ROW_CLASSES - 1;
}
__device__ __forceinline__ int32_t row_scale(int shift) {
    const int c = row_class(shift);
    return c << 16 | __builtin_bit_cast(uint16_t, (half_t)ldexpf(1.0f, shift + 16 * c));
}
struct RowScales {
    const int32_t *scales;   // of the operand's row ok0
    const int32_t *sums;     // binades that the row sums of a are to be taken by (not the product: it is in `scales`), or NULL
    int cls;
    // which of sixteen rows is lane half h's e-th value; perm: GemmOperand's
    static __device__ __forceinline__ constexpr int at(int e, int h, int perm) { return perm ? (e & 3) + 8 * (e >> 2) + 4 * h : 8 * h + e; }
};
// sixteen words at a wave-uniform address, by scalar loads
struct Row16 { int32_t v[16]; };
__device__ __forceinline__ Row16 row16(const int32_t *p, int row) {
    typedef const __attribute__((address_space(4))) int32_t *Constant;
    const Constant c = (Constant)(p + __builtin_amdgcn_readfirstlane(row));
    Row16 r;
#pragma unroll
    for (int k = 0; k < 16; ++k) r.v[k] = c[k];
    return r;
}

struct GemmOperand {
    const half_t *p;     // panel 0, row 0
    int64_t rows;        // rows of a panel (a multiple of 256)
    int perm;            // KS: bits 2 and 3 of the row index change places (the order in which G's columns are stored)
};

// One operand's tile of BR rows (KC) / BR columns (KS).
template <bool KS, bool SPLIT, int BR, int NW> struct TileStage {
    static constexpr int INSTR = BR / 16 / NW;                     // 1 KB wave instructions per wave and step: 16 rows of a panel each
    static_assert(BR / 16 % NW == 0, "tile rows must spread evenly over the waves");
    static constexpr int KSTEP = SPLIT ? 16 : 32;                  // k values per step = columns per panel
    const half_t *base;
    int64_t advance;                                               // elements per step
    uint32_t off[INSTR];

    // KC: tile rows [r0, r0 + BR), k from panel k0.  KS: tile columns from panel c0 (the last of `panels` again beyond), k from row k0.
    __device__ __forceinline__ void init(const GemmOperand &o, int64_t r0, int64_t panel, int panels_left, int wave, int lane) {
        base = o.p + (panel * o.rows + r0) * 32;
        advance = KS ? KSTEP * 32 : o.rows * 32;
#pragma unroll
        for (int j = 0; j < INSTR; ++j) {
            const int q = wave + j * NW;
            if (!KS) {
                const int r = q * 16 + (lane >> 2);
                off[j] = r * 32 + ((lane & 3) ^ ((r >> 2) & 3)) * 8;
            } else {
                int pan = SPLIT ? q : q >> 1, r = (SPLIT ? 0 : (q & 1) * 16) + (lane >> 2), ch = lane & 3;
                if (SPLIT) ch ^= (pan & 1) << 1;
                if (o.perm) r = (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1);
                pan = pan < panels_left ? pan : panels_left - 1;
                off[j] = (uint32_t)(pan * o.rows * 32) + r * 32 + ch * 8;
            }
        }
    }
    __device__ __forceinline__ void load(int step, int64_t plane, char *lds, int wave) const {
        const half_t *b = base + step * advance + plane;
#pragma unroll
        for (int j = 0; j < INSTR; ++j)
            __builtin_amdgcn_global_load_lds((const TNP_GLB void *)(b + off[j]), (TNP_LDS void *)(lds + (wave + j * NW) * 1024), 16, 0, 0);
    }
    // KC: operand of one 32-row block at tile row r0, sub-step ss of 16 values, plane 0 = hi / 1 = lo (SPLIT)
    static __device__ __forceinline__ half8 frag(const char *lds, int r0, int ss, int plane, int lane) {
        const int r = r0 + (lane & 31), ch = (SPLIT ? plane : ss) * 2 + (lane >> 5);
        return *(const half8 *)(lds + r * 64 + ((ch ^ ((r >> 2) & 3)) * 16));
    }
    // KS: LDS byte address of the first value this lane fetches for 32 columns from c, k rows 0 .. 3 of its half; rows row + 4 and row + 16
    // are constant offsets
    static constexpr int ROW4 = 4 * 64, ROW16 = 16 * 64;
    static __device__ __forceinline__ uint32_t ks_addr(const char *lds, int c, int plane, int lane) {
        const int g = lane >> 4, j = lane & 15, row = 8 * (g >> 1) + (j >> 2);
        int at;
        if (SPLIT) at = ((c >> 4) + (g & 1)) * 1024 + row * 64 + (plane ^ (g & 1)) * 32 + (j & 3) * 8;      // c is a multiple of 32
        else at = (c >> 5) * 2048 + row * 64 + (g & 1) * 32 + (j & 3) * 8;
        return (uint32_t)(uintptr_t)(TNP_LDS const char *)lds + at;
    }
};

// 32-column blocks of KS tiles at the LDS addresses a[], k rows 0 .. 3 and (R4 bytes on) 4 .. 7 of every half.  One asm block that ends
// with its own wait: as builtins these reads would first wait for every global_load_lds in flight, that is for the tiles of the
// next steps.


template <int R4> __device__ __forceinline__ void ks_read(const uint32_t (&a)[2], half8 (&f)[2]) {
    int2v r[4];
    asm volatile(
                 "ds_read_b64_tr_b16 %0, %4\n\t"
                 "ds_read_b64_tr_b16 %1, %4 offset:%c6\n\t"
                 "ds_read_b64_tr_b16 %2, %5\n\t"
                 "ds_read_b64_tr_b16 %3, %5 offset:%c6\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
                 : "v"(a[0]), "v"(a[1]), "i"(R4)
                 : "memory");
#pragma unroll
    for (int k = 0; k < 2; ++k) f[k] = __builtin_bit_cast(half8, int4v{r[2 * k].x, r[2 * k].y, r[2 * k + 1].x, r[2 * k + 1].y});
}
template <int R4> __device__ __forceinline__ void ks_read(const uint32_t (&a)[4], half8 (&f)[4]) {
    int2v r[8];
    asm volatile(
                 "ds_read_b64_tr_b16 %0, %8\n\t"
                 "ds_read_b64_tr_b16 %1, %8 offset:%c12\n\t"
                 "ds_read_b64_tr_b16 %2, %9\n\t"
                 "ds_read_b64_tr_b16 %3, %9 offset:%c12\n\t"
                 "ds_read_b64_tr_b16 %4, %10\n\t"
                 "ds_read_b64_tr_b16 %5, %10 offset:%c12\n\t"
                 "ds_read_b64_tr_b16 %6, %11\n\t"
                 "ds_read_b64_tr_b16 %7, %11 offset:%c12\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "i"(R4)
                 : "memory");
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = __builtin_bit_cast(half8, int4v{r[2 * k].x, r[2 * k].y, r[2 * k + 1].x, r[2 * k + 1].y});
}
template <int R4> __device__ __forceinline__ void ks_read(const uint32_t (&a)[8], half8 (&f)[8]) {
    int2v r[16];
    asm volatile(
                 "ds_read_b64_tr_b16 %0, %16\n\t"
                 "ds_read_b64_tr_b16 %1, %16 offset:%c24\n\t"
                 "ds_read_b64_tr_b16 %2, %17\n\t"
                 "ds_read_b64_tr_b16 %3, %17 offset:%c24\n\t"
                 "ds_read_b64_tr_b16 %4, %18\n\t"
                 "ds_read_b64_tr_b16 %5, %18 offset:%c24\n\t"
                 "ds_read_b64_tr_b16 %6, %19\n\t"
                 "ds_read_b64_tr_b16 %7, %19 offset:%c24\n\t"
                 "ds_read_b64_tr_b16 %8, %20\n\t"
                 "ds_read_b64_tr_b16 %9, %20 offset:%c24\n\t"
                 "ds_read_b64_tr_b16 %10, %21\n\t"
                 "ds_read_b64_tr_b16 %11, %21 offset:%c24\n\t"
                 "ds_read_b64_tr_b16 %12, %22\n\t"
                 "ds_read_b64_tr_b16 %13, %22 offset:%c24\n\t"
                 "ds_read_b64_tr_b16 %14, %23\n\t"
                 "ds_read_b64_tr_b16 %15, %23 offset:%c24\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]), "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]), "=&v"(r[15])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]), "i"(R4)
                 : "memory");
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = __builtin_bit_cast(half8, int4v{r[2 * k].x, r[2 * k].y, r[2 * k + 1].x, r[2 * k + 1].y});
}

// Waits until at most N of this wave's loads are in flight and all its LDS reads are done, then meets the other waves.
template <int N> __device__ __forceinline__ void stage_barrier() {
    asm volatile("s_waitcnt vmcnt(%c0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

__device__ __forceinline__ void stage_barrier_only() { asm volatile("s_barrier" ::: "memory"); }

// All of a wave's operand blocks of one step: NB blocks of 32 rows (KC) / columns (KS) from c, each with two 8-value registers (the two
// sub-steps of 16 values, or the hi and lo planes of a split step): f[2 * block + which].
template <typename ST, bool KS, bool SPLIT, int NB>
__device__ __forceinline__ void step_frags(const char *lds, int c, int lane, half8 (&f)[2 * NB]) {
    if constexpr (KS) {
        uint32_t a[2 * NB];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int w = 0; w < 2; ++w) a[2 * b + w] = ST::ks_addr(lds, c + b * 32, SPLIT ? w : 0, lane) + (SPLIT ? 0 : w * ST::ROW16);
        ks_read<ST::ROW4>(a, f);
    } else {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int w = 0; w < 2; ++w) f[2 * b + w] = ST::frag(lds, c + b * 32, w, w, lane);
    }
}

template <bool SPLIT, int TM, int TN>
__device__ __forceinline__ void step_mfma(const half8 (&fa)[2 * TM], const half8 (&fb)[2 * TN], f32x16 (&acc)[TM][TN]) {
    // products per block pair: the two sub-steps, or lo * hi, hi * lo, hi * hi (the small ones are not lost against the large)
    constexpr int N = SPLIT ? 3 : 2;
    constexpr int wa[3] = {SPLIT ? 1 : 0, SPLIT ? 0 : 1, 0}, wb[3] = {0, 1, 0};
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[2 * i + wa[k]], fb[2 * j + wb[k]], acc[i][j], 0, 0, 0);
}

// sums over k of an operand's values, per row of the block: asum[i] += what this lane holds of block i (half of the k values; the
// other half of the wave holds the rest)
template <int TM> __device__ __forceinline__ void step_row_sums(const half8 (&fa)[2 * TM], float (&asum)[TM]) {
    typedef half_t half2v __attribute__((ext_vector_type(2)));
    const half2v one = {(half_t)1.0f, (half_t)1.0f};
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                asum[i] = __builtin_amdgcn_fdot2(half2v{fa[2 * i + w][2 * e], fa[2 * i + w][2 * e + 1]}, one, asum[i], false);
}

// a step's words; row: of the step's first k value
template <bool SPLIT, bool SUMS> struct StepWords {
    static constexpr int N = SPLIT ? 1 : 2;
    Row16 scales[N], sums[SUMS ? N : 1];
    __device__ __forceinline__ void load(const RowScales &rs, int row) {
#pragma unroll
        for (int w = 0; w < N; ++w) scales[w] = row16(rs.scales, row + 16 * w);
        if (SUMS && rs.sums)
#pragma unroll
            for (int w = 0; w < N; ++w) sums[SUMS ? w : 0] = row16(rs.sums, row + 16 * w);
    }
};

// One step's KS operand times its rows' scales
template <bool SPLIT, bool PERM, int NB, typename Words>
__device__ __forceinline__ void step_scale(half8 (&f)[2 * NB], const RowScales &rs, const Words &words, int lane) {
#pragma unroll
    for (int w = 0; w < (SPLIT ? 1 : 2); ++w) {
        __builtin_amdgcn_sched_barrier(0);                           // sixteen rows at a time: more of them spill registers
        const Row16 &r = words.scales[w];
        uint32_t bits[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) bits[k] = r.v[k] >> 16 == rs.cls ? r.v[k] & 0xffff : 0;
        int4v sc;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const uint32_t low = bits[RowScales::at(e, 0, PERM)] | bits[RowScales::at(e + 1, 0, PERM)] << 16,
                           high = bits[RowScales::at(e, 1, PERM)] | bits[RowScales::at(e + 1, 1, PERM)] << 16;
            sc[e / 2] = lane >> 5 ? high : low;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int p = 0; p < (SPLIT ? 2 : 1); ++p) f[2 * b + (SPLIT ? p : w)] *= __builtin_bit_cast(half8, sc);
    }
}

// the sums of step_row_sums over the rows of one class, each by the binades that its sums are to be taken by
template <bool SPLIT, int TM, typename Words>
__device__ __forceinline__ void step_row_sums(const half8 (&fa)[2 * TM], float (&asum)[TM], const RowScales &rs, const Words &words, int lane) {
#pragma unroll
    for (int w = 0; w < (SPLIT ? 1 : 2); ++w) {
        __builtin_amdgcn_sched_barrier(0);
        const Row16 &r = words.scales[w];
        float by[16];
        if (rs.sums) {
            const Row16 &n = words.sums[w];
#pragma unroll
            for (int k = 0; k < 16; ++k) by[k] = r.v[k] >> 16 == rs.cls && n.v[k] > -127 ? __uint_as_float((uint32_t)(127 + n.v[k]) << 23) : 0.0f;
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) by[k] = r.v[k] >> 16 == rs.cls ? 1.0f : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float b = lane >> 5 ? by[8 + e] : by[e];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                asum[i] = fmaf((float)fa[2 * i + w][e], b, asum[i]);
                if (SPLIT) asum[i] = fmaf((float)fa[2 * i + 1][e], b, asum[i]);
            }
        }
    }
}

// The steps of [s0, s1) from the first to the last that has a row of the class, the same for all lanes.
template <int KSTEP> __device__ __forceinline__ void class_steps(const RowScales &rs, int wrap, int &s0, int &s1, int lane) {
    if (rs.cls == 0 || (s0 < wrap && s1 > wrap)) return;             // most rows' class, or both planes of the other operand: all of them
    const int back = s0 >= wrap ? wrap : 0, end = (s1 - back) * KSTEP;
    int first = INT32_MAX, last = -1;
    constexpr int U = 16;                                            // words in flight
    for (int r0 = (s0 - back) * KSTEP + lane; r0 < end; r0 += 64 * U) {
        int32_t v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = rs.scales[r0 + u * 64 < end ? r0 + u * 64 : r0];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * 64;
            if (r >= end || v[u] >> 16 != rs.cls) continue;
            first = first < r ? first : r;
            last = r;
        }
    }
    for (int o = 32; o; o >>= 1) {
        const int f = __shfl_xor(first, o), l = __shfl_xor(last, o);
        first = first < f ? first : f;
        last = last > l ? last : l;
    }
    first = __builtin_amdgcn_readfirstlane(first);
    last = __builtin_amdgcn_readfirstlane(last);
    s1 = last < 0 ? s0 : back + last / KSTEP + 1;
    s0 = last < 0 ? s0 : back + first / KSTEP;
}

// One workgroup's products: init() takes the tile at (row ar, panel ap) of a and (br, bp) of b (al / bl: panels from there to the last,
// KS), first() starts to fetch its steps [s0, s1), run() accumulates them into acc.  After run() the ring is free: first() of the next
// tile (a_rows() moves a KC operand a on by whole rows) can be called before this one's results are used, which hides its latency.
// LDS: NST * (BM + BN) * 64 bytes.
//
// Eight waves (two per SIMD) take turns: while one half of the workgroup fetches the operands of a step into registers, the other
// half multiplies the step it has fetched; a barrier per turn keeps them half a step apart.  In lockstep both waves of a SIMD would
// fetch at the same time and leave the matrix cores idle meanwhile (2150 cycles per step of 1024 cycles of matrix work).  With
// four waves the other workgroups on the CU fill that time.
//
// SUMS: with `sums` (the same for the wave), asum[] gathers the row sums of a as well (step_row_sums).
//
// An unsplit a may have a second plane, `plane` elements behind the first: the steps from `wrap` on run over it, with b's steps from the
// first one again.
//
// SCALED: b's rows on scales of their own (RowScales), in G's stored order of them where a is read as KC; acc is added to, not set.
template <bool SPLIT, bool A_KS, bool B_KS, int BM, int BN, int WM, int WN, int NST> struct TileGemm {
    static constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, STAGE = (BM + BN) * 64;
    static constexpr bool TURNS = NW == 8;
    typedef TileStage<A_KS, SPLIT, BM, NW> SA;
    typedef TileStage<B_KS, SPLIT, BN, NW> SB;
    static constexpr int LOADS = SA::INSTR + SB::INSTR;            // per wave and step
    static_assert(NST >= 3, "the tile after next is in flight while one is read");
    SA sa;
    SB sb;
    char *lds;
    int lane, wave, wrap;
    int64_t plane;

    __device__ __forceinline__ void init(const GemmOperand &a, const GemmOperand &b, int64_t ar, int64_t ap, int al, int64_t br, int64_t bp, int bl,
                                         char *lds_) {
        lds = lds_;
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wrap = INT32_MAX;
        plane = 0;
        sa.init(a, ar, ap, al, wave, lane);
        sb.init(b, br, bp, bl, wave, lane);
    }
    __device__ __forceinline__ void a_rows(int rows) { sa.base += (int64_t)rows * 32; }
    __device__ __forceinline__ void two_planes(int64_t plane_, int wrap_) { plane = plane_; wrap = wrap_; }
    __device__ __forceinline__ void load(int s, int stage) {
        const bool second = s >= wrap;
        const int k = second ? s - wrap : s;
        sa.load(k, second ? plane : 0, lds + stage * STAGE, wave);
        sb.load(k, 0, lds + stage * STAGE + BM * 64, wave);
    }
    __device__ __forceinline__ void first(int s0, int s1) {
#pragma unroll
        for (int k = 0; k < NST - 1; ++k)
            if (s0 + k < s1) load(s0 + k, k);
    }
    // the step that has `left` steps behind it has landed in every wave: at most NST - 2 steps' loads are still in flight
    template <int N = NST - 2> static __device__ __forceinline__ void landed(int left) {
        if constexpr (N > 0) {
            if (left >= N) stage_barrier<N * LOADS>();
            else landed<N - 1>(left);
        } else {
            stage_barrier<0>();
        }
    }
    static __device__ __forceinline__ void clear(f32x16 (&acc)[TM][TN]) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    }
    template <bool SUMS, bool SCALED>
    __device__ __forceinline__ void run(int s0, int s1, f32x16 (&acc)[TM][TN], bool sums, float (&asum)[TM], const RowScales &rs) {
        const int wm = wave / WN, wn = wave % WN;
        if (!SCALED) clear(acc);
        if (s0 >= s1) return;
        landed(s1 - 1 - s0);
        if (TURNS && wave >= 4) stage_barrier_only();
        int cur = 0;
        half8 fa[2 * TM], fb[2 * TN];
        auto row = [&](int s) { return (s < wrap ? s : s - wrap) * SB::KSTEP; };
        StepWords<SPLIT, SUMS> words;
        if constexpr (SCALED) words.load(rs, row(s0));
        for (int s = s0; s < s1; ++s) {
            const char *la = lds + cur * STAGE, *lb = la + BM * 64;
            step_frags<SB, B_KS, SPLIT, TN>(lb, wn * TN * 32, lane, fb);
            step_frags<SA, A_KS, SPLIT, TM>(la, wm * TM * 32, lane, fa);
            if constexpr (SCALED) step_scale<SPLIT, !A_KS, TN>(fb, rs, words, lane);
            if (s + NST - 1 < s1) load(s + NST - 1, cur == 0 ? NST - 1 : cur - 1);   // the buffer that every wave left one barrier ago
            cur = cur + 1 == NST ? 0 : cur + 1;
            if (TURNS) {
                __builtin_amdgcn_sched_barrier(0);
                if (s + 1 < s1) landed(s1 - 2 - s); else stage_barrier<0>();
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
                step_mfma<SPLIT, TM, TN>(fa, fb, acc);
                if (SUMS && sums) {
                    if constexpr (SCALED) step_row_sums<SPLIT, TM>(fa, asum, rs, words, lane);
                    else step_row_sums<TM>(fa, asum);
                }
                if constexpr (SCALED) words.load(rs, row(s + 1 < s1 ? s + 1 : s));
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
                stage_barrier_only();
                __builtin_amdgcn_sched_barrier(0);
            } else {
                step_mfma<SPLIT, TM, TN>(fa, fb, acc);
                if (SUMS && sums) {
                    if constexpr (SCALED) step_row_sums<SPLIT, TM>(fa, asum, rs, words, lane);
                    else step_row_sums<TM>(fa, asum);
                }
                if constexpr (SCALED) words.load(rs, row(s + 1 < s1 ? s + 1 : s));
                landed(s1 - 2 - s);                                // after the last step: every wave is done with the ring
            }
        }
        if (TURNS && wave < 4) stage_barrier_only();
    }
};

// Workgroup -> tile: the eight XCDs take the workgroups in turn, so each gets a contiguous share of the tiles, walked in groups of
// eight tile rows; the panels of a group stay in the XCD's own L2.  Returns false for the workgroups behind the last tile.
__device__ __forceinline__ bool gemm_tile_of(int bid, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int total = tiles_m * tiles_n, per = (total + 7) / 8;
    const int t = (bid & 7) * per + (bid >> 3);
    if ((bid >> 3) >= per || t >= total) return false;
    const int width = 8 * tiles_n, g = t / width, first = g * 8;
    const int h = tiles_m - first < 8 ? tiles_m - first : 8, r = t - g * width;
    tm = first + r % h;
    tn = r / h;
    return true;
}
inline int gemm_grid(int64_t tiles) { return (int)((tiles + 7) / 8 * 8); }

}  // namespace tnp
