// Cross entropy over a vocabulary (gfx950): the output layer and its softmax loss as one operator,
//     l_iv = hidden_i . weight_v + bias_v,   lse_i = log sum_v exp(l_iv),   loss_i = lse_i - l_i,target(i)
//     G_iv = g_i (exp(l_iv - lse_i) - [v == target(i)]),   dhidden = G weight,   dweight = G^T hidden,   dbias_v = sum_i G_iv
// The logits are never kept: the forward pass leaves per row the running maximum and sum of every vocabulary tile, the backward
// pass forms the logits again, piece by piece of the vocabulary, as G in fp16 (twice fp16 for fp32 and fp16 inputs), which both gradient
// products read.  Forming them again costs 2 M D V operations; writing, reading and correcting the fp32 logits would cost 12 bytes
// each, more than that for every D below about 2000.
//
// Numbers.  Inputs are packed once per call as fp16 times one power of two per tensor, so that its largest element lies in
// [2^14, 2^15); a row whose largest element is below 2^-16 of that gets a power of two of its own (a "far" row), so that no row's bits go by
// another's size.  bf16 and fp16 values are exact down to 2^-12 of their row's largest, fp32 values become two fp16 numbers (vocab_gemm.h); an error of
// 2^-23 of the value or of its row's largest, usually 2^-40 of the latter.  Logits of far rows or entries get their powers of two one by one;
// the gradient products, where rows are summed over, take far rows in classes (vocab_gemm.h), one run each.  G = 2^15 (g_i / max g) (p - y),
// with a power of two per row instead of 1 / max g where the row's upstream gradient is below 2^-18 of the largest, is rounded to fp16 for
// bf16 gradients (11 bits, eight times finer than what they are rounded to: their error grows by less than a hundredth) and to two fp16
// numbers for fp32 and fp16 ones (one of them would be as coarse as the fp16 gradient itself).  All sums, maxima and statistics are fp32; the sum of the losses is fp64.
//
// A negative target marks an absent row: its hidden state is not read (it may be NaN), its loss and gradients are zero.  Packing leaves
// the absent rows out, so that everything behind it runs on the rows that are there (a fifth of a crowd's tracks are absent, more
// where only some are predicted); their number stays on the device, launches are sized for all rows and the workgroups behind the
// last row end at once.  A target >= V is an error that shows: NaN loss, NaN gradients.
#include "vocab_gemm.h"
#include "../../include/trajnet_hip_profile.h"

#include <math.h>

#include <algorithm>

namespace tnp {

static constexpr float CE_LOG2E = 1.4426950408889634f;
static constexpr double CE_LN2 = 0.6931471805599453;
static constexpr float CE_NEG_INF = -__builtin_inff();
static constexpr int CE_AMAX_BLOCKS = 512;            // per tensor, the hidden states in as many shares of rows as they are packed in
static constexpr int CE_ROW_PAD = 256, CE_COL_PAD = 256;
// Groups of 16 entries that a wave scores at a time for more than 16 rows, from this vocabulary on (more than one wave per SIMD with one):
// 64 x 65536 x 512 bf16 37 us against 48, 64 x 20480 x 512 bf16 25 against 29; 64 x 16384 x 128 fp32 21 against 16
static constexpr int CE_SCORE_GROUPS = 2, CE_SCORE_GROUPS_FROM = 20480;
static constexpr int CE_JOIN_BLOCKS = 1 << 20;         // a grid holds fewer than 2^32 threads
// rows up to which scoring reads the inputs in place: 64 x 65536 x 512 bf16 37 us against 62 packed, fp32 74 against 127
static constexpr int CE_SCORE_ROWS = 64;

// G as two fp16 numbers: panels of both (SPLIT operands), or one plane of panels behind the other
template <typename T, bool SPLIT> static constexpr bool CE_TWO_PLANES = !SPLIT && std::is_same<T, half_t>::value;
static inline int ce_g_planes(int dtype) { return dtype == TNP_BF16 ? 1 : 2; }

struct CeScalars {            // head of the saved area
    int ex, ew;               // packed = value * 2^-e
    uint32_t ticket;          // last-workgroup counter of the loss sum
    int live;                 // rows that are there
    uint32_t x_classes, w_classes;      // bit c: rows of class c (vocab_gemm.h) among the hidden states, the weight
};
static constexpr int CE_FAR = 16;      // binades below the tensor's largest element from which on a row has its own scale
struct CeUpstream {           // reduction none, head of the backward pass's workspace
    float gmax;               // largest finite |grad| of the rows that are there, 1 where that is 0
    uint32_t classes;         // bit c: rows of class c, by their hidden state's scale and their gradient's together
};
__device__ __forceinline__ int ce_padded(int live) { return (live + 255) & ~255; }

struct CeShape {
    int64_t M, Mp;            // rows, padded to 256
    int V, Vp, D;             // vocabulary, padded to 256
    int split;                // fp32: two planes
    int panels;               // of 32 columns (16 split ones): k steps of the logits
};

// ---- scales and packing -----------------------------------------------------------------------------------------------------
// largest finite |element| of rows [r0, r1): the rows' accesses one after the other, four in flight per lane.  16384 + 65536 rows of 1024 bf16:
// 38 us, 4.4 TB/s; packing them reads from the caches behind it: 57 us for 168 MB in and as much out
template <typename T, int VE>
__device__ __forceinline__ float ce_rows_amax(const T *x, int64_t ld, int64_t r0, int64_t r1, const int64_t *target, int D) {
    const uint32_t per = (uint32_t)D / VE, n = (uint32_t)(r1 - r0) * per;
    float a = 0.0f;
    constexpr int U = 4;
    for (uint32_t k = threadIdx.x; k < n; k += 256 * U) {
        Pack<T, VE> p[U];
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t q = k + u * 256, row = q / per, c = q - row * per;
            in[u] = q < n;                                       // behind the end: the first row again, loads under a condition wait
            const int64_t r = r0 + (in[u] ? row : 0);            // for each other
            if (target) in[u] = in[u] && target[r] >= 0;
            p[u] = *(const Pack<T, VE> *)(x + r * ld + (q < n ? c * VE : 0));
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float v = fabsf(to_f32(p[u].v[e]));
                a = fmaxf(a, in[u] && v < __builtin_inff() ? v : 0.0f);      // infinities and NaN do not set the scale
            }
    }
    return a;
}

template <typename T, int VX, int VW>
__global__ void __launch_bounds__(256) ce_amax_kernel(const T *x, int64_t ldx, int64_t M, const int64_t *target, const T *w, int64_t ldw, int V,
                                                      int D, int x_blocks, float *part, int *count, CeScalars *sc) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool is_w = blockIdx.x >= CE_AMAX_BLOCKS;
    const int64_t bid = is_w ? blockIdx.x - CE_AMAX_BLOCKS : blockIdx.x, rows = is_w ? V : M, blocks = is_w ? CE_AMAX_BLOCKS : x_blocks;
    const int64_t r0 = bid < blocks ? rows * bid / blocks : rows, r1 = bid < blocks ? rows * (bid + 1) / blocks : rows;
    float a = is_w ? ce_rows_amax<T, VW>(w, ldw, r0, r1, nullptr, D) : ce_rows_amax<T, VX>(x, ldx, r0, r1, target, D);
    __shared__ float sh[4];
    if (!is_w) {
        __shared__ int n[4];
        int c = 0;
        for (int64_t r = r0 + threadIdx.x; r < r1; r += 256) c += target[r] >= 0;
        for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o);
        if (lane == 0) n[wave] = c;
        __syncthreads();
        if (threadIdx.x == 0) count[bid] = n[0] + n[1] + n[2] + n[3];
    }
    for (int o = 32; o; o >>= 1) a = fmaxf(a, __shfl_xor(a, o));
    if (lane == 0) sh[wave] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        part[blockIdx.x] = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
        if (blockIdx.x == 0) {
            sc->ticket = 0;
            sc->x_classes = sc->w_classes = 1;
        }
    }
}

// exponent e with max |x| * 2^-e in [2^14, 2^15); 0 for an all-zero tensor
__device__ __forceinline__ int ce_exponent(float a) {
    if (a == 0.0f) return 0;
    int e;
    frexpf(a, &e);
    return e - 15;
}

// sixteen rows into panels (vocab_gemm.h): lane = (row, 16-byte chunk), so a panel is written as one contiguous kilobyte.  This lane's
// row: src row `from` (negative: zeros) to dst row `to` (negative: nothing), times 2^-e.  Returns the largest finite |element| that this lane has seen.
template <typename T, int VE, bool SPLIT>
__device__ __forceinline__ float ce_pack_rows_at(const T *src, int64_t ld, int64_t from_row, int64_t to, int D, int e, half_t *dst,
                                                 int64_t panel_rows, int panels, int lane) {
    constexpr int NV = 8;                                        // values per chunk; a split chunk is the hi or the lo half of eight
    const bool live = from_row >= 0;
    const int ch = lane & 3, c0 = SPLIT ? (ch & 1) * 8 : ch * 8;
    constexpr int U = 4;                                         // panels in flight
    const T *from = src + (live ? from_row : 0) * ld;                 // rows and columns that are not there: row 0, column 0, not used
    half_t *out = dst + (to < 0 ? 0 : to) * 32 + ch * 8;
    float top = 0.0f;
    for (int p = 0; p < panels; p += U) {
        Pack<T, VE> q[U][NV / VE];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < NV / VE; ++k) {
                const int c = (p + u) * (SPLIT ? 16 : 32) + c0 + k * VE;
                q[u][k] = *(const Pack<T, VE> *)(from + (c < D ? c : 0));
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p + u >= panels) break;
            half8 o;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const bool there = live && (p + u) * (SPLIT ? 16 : 32) + c0 + k < D;
                const float x = there ? to_f32(q[u][k / VE].v[k % VE]) : 0.0f, v = ldexpf(x, -e);
                const half_t hi = (half_t)v;
                // an infinity is the lo half, beside a hi of zero: it meets the other operand's hi alone, whose sign is the value's
                const bool inf = SPLIT && fabsf(v) == __builtin_inff();
                o[k] = SPLIT && ch >= 2 ? (inf ? hi : (half_t)(v - (float)hi)) : inf ? (half_t)0.0f : hi;
                top = fmaxf(top, fabsf(x) < __builtin_inff() ? fabsf(x) : 0.0f);
            }
            if (to >= 0) *(half8 *)(out + (p + u) * panel_rows * 32) = o;
        }
    }
    return top;
}

// classes |= the wave's bits: one atomic per wave, none where they are there already
__device__ __forceinline__ void ce_add_classes(uint32_t *classes, uint32_t bits) {
    for (int o = 32; o; o >>= 1) bits |= __shfl_xor(bits, o);
    if ((threadIdx.x & 63) == 0 && (bits & ~__hip_atomic_load(classes, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))) atomicOr(classes, bits);
}

// the same on the tensor's exponent e, and once more on their own the rows that are far below it; exps[to], scales[to]: the row's exponent
// and its word for the gradient products
template <typename T, int VE, bool SPLIT>
__device__ __forceinline__ void ce_pack_rows(const T *src, int64_t ld, int64_t from_row, int64_t to, int D, int e, half_t *dst, int64_t panel_rows,
                                             int panels, int lane, int32_t *exps, int32_t *scales, uint32_t *classes) {
    float top = ce_pack_rows_at<T, VE, SPLIT>(src, ld, from_row, to, D, e, dst, panel_rows, panels, lane);
    top = fmaxf(top, __shfl_xor(top, 1));                        // the row's four lanes
    top = fmaxf(top, __shfl_xor(top, 2));
    const int own = ce_exponent(top);
    const bool far = top > 0.0f && own < e - CE_FAR;
    if (to >= 0 && (lane & 3) == 0) {
        exps[to] = far ? own : e;
        scales[to] = row_scale(far ? own - e : 0);
    }
    if (!__any(far)) return;
    ce_pack_rows_at<T, VE, SPLIT>(src, ld, from_row, far ? to : -1, D, own, dst, panel_rows, panels, lane);
    ce_add_classes(classes, far && to >= 0 ? 1u << row_class(own - e) : 0);
}

template <typename T, int VX, int VW, bool SPLIT>
__global__ void __launch_bounds__(256) ce_pack_kernel(const T *x, int64_t ldx, const int64_t *target, const T *w, int64_t ldw, CeShape sh,
                                                      const float *part, const int *count, CeScalars *sc, half_t *xp, half_t *wp, int32_t *orig,
                                                      int32_t *tc, int32_t *xe, int32_t *xs, int32_t *we, int32_t *ws, int x_blocks) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = threadIdx.x;
    const bool is_w = (int)blockIdx.x >= x_blocks;
    __shared__ float red[4];
    __shared__ int2 cnt[4];
    __shared__ int32_t list[256];
    float a = fmaxf(part[(is_w ? CE_AMAX_BLOCKS : 0) + tid], part[(is_w ? CE_AMAX_BLOCKS : 0) + 256 + tid]);
    // rows that are there: those of the shares before this one, all of them
    int2 n = make_int2(0, 0);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int c = count[k * 256 + tid];
        n.x += k * 256 + tid < (int)blockIdx.x ? c : 0;
        n.y += c;
    }
    for (int o = 32; o; o >>= 1) {
        a = fmaxf(a, __shfl_xor(a, o));
        n.x += __shfl_xor(n.x, o);
        n.y += __shfl_xor(n.y, o);
    }
    if (lane == 0) { red[wave] = a; cnt[wave] = n; }
    __syncthreads();
    const int e = ce_exponent(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    if (is_w) {
        if (tid == 0 && (int)blockIdx.x == x_blocks) sc->ew = e;
        const int blocks = gridDim.x - x_blocks;
        for (int64_t r = ((int)blockIdx.x - x_blocks) * 64 + wave * 16 + (lane >> 2); r < sh.Vp; r += blocks * 64)
            ce_pack_rows<T, VW, SPLIT>(w, ldw, r < sh.V ? r : -1, r, sh.D, e, wp, sh.Vp, sh.panels, lane, we, ws, &sc->w_classes);
        return;
    }
    int base = cnt[0].x + cnt[1].x + cnt[2].x + cnt[3].x;
    const int live = cnt[0].y + cnt[1].y + cnt[2].y + cnt[3].y;
    if (tid == 0 && blockIdx.x == 0) { sc->ex = e; sc->live = live; }
    const int64_t r0 = sh.M * (int64_t)blockIdx.x / x_blocks, r1 = sh.M * (int64_t)(blockIdx.x + 1) / x_blocks;
    for (int64_t rc = r0; rc < r1; rc += 256) {
        // the next 256 rows' list of those that are there
        const int64_t t = rc + tid < r1 ? target[rc + tid] : -1;
        const uint64_t m = __ballot(t >= 0);
        __syncthreads();                                         // list and cnt of the rows before are done with
        if (lane == 0) cnt[wave].x = __popcll(m);
        __syncthreads();
        int at = 0, num = 0;
        for (int k = 0; k < 4; ++k) {
            at += k < wave ? cnt[k].x : 0;
            num += cnt[k].x;
        }
        at += __popcll(m & ((1ull << lane) - 1));
        if (t >= 0) {
            list[at] = (int32_t)(rc + tid);
            orig[base + at] = (int32_t)(rc + tid);
            tc[base + at] = t < sh.V ? (int32_t)t : sh.V;        // V: no such target
        }
        __syncthreads();
        for (int g = wave * 16; g < num; g += 64) {
            const int i = g + (lane >> 2);
            ce_pack_rows<T, VX, SPLIT>(x, ldx, i < num ? list[i] : -1, i < num ? base + i : -1, sh.D, e, xp, sh.Mp, sh.panels, lane, xe, xs,
                                        &sc->x_classes);
        }
        base += num;
    }
    // zero rows up to the next multiple of 256
    for (int64_t r = live + (int64_t)blockIdx.x * 64 + wave * 16 + (lane >> 2); r - (lane >> 2) < ce_padded(live); r += (int64_t)x_blocks * 64)
        ce_pack_rows<T, VX, SPLIT>(x, ldx, -1, r < ce_padded(live) ? r : -1, sh.D, e, xp, sh.Mp, sh.panels, lane, xe, xs, &sc->x_classes);
}

// ---- logits: statistics forward, G backward ---------------------------------------------------------------------------------
// The vocabulary runs over the rows of the matrix instruction, so a lane holds 16 logits of ONE hidden row per 32 x 32 block and
// maxima, sums and exponentials stay inside the lane; the two halves of a wave meet once per share of the vocabulary.  16384 x 65536 x 1024
// bf16: 2.05 ms of statistics (1.07 PFLOP/s), 2.18 with G written (2 GB); 4096 x 16384 x 512 fp32: 179 and 209 us (384 and 329 TFLOP/s; a
// library product in fp32: 138).  The matrix pipe is busy for 53 to 64 % of the cycles, at 1.9 GHz; the exponentials of a tile, three
// vector instructions per matrix instruction, and its barriers take the rest.
struct CeLogits {
    GemmOperand w, x;
    const CeScalars *sc;
    const int32_t *tc, *orig; // of the rows that are there: target (V: none such), row of the caller
    const int32_t *xe, *we;   // exponents of hidden rows and vocabulary entries
    int64_t Mp;
    int V, v0, tiles_v, v_shares, steps;
    // forward
    float2 *part;             // [vocabulary share, wave row][Mp]: (max, sum of 2^(l - max)), base 2
    float *tlogit;            // [Mp] target's logit, base 2
    // backward
    const float2 *stat;       // [Mp] (largest logit, base 2; 1 / sum of 2^(l - largest)), padding (+inf, 0), no such target (.., NaN)
    const float *grad;        // reduction none: [M]
    CeUpstream *up;           // ... what is known of it
    int32_t *gs, *xs;         // ... binades [Mp] by which a row of G lies below the largest gradient's scale, words of these and the hidden states' together
    half_t *g;                // panels of Mp rows, column 0 = vocabulary entry v0
    int64_t g_plane;          // elements from a plane of G to the next
};

// bias in base 2; a finite one stays finite (the lowest value of fp32 as a mask: where it masks a whole row, all entries are alike)
template <typename T> __device__ __forceinline__ float ce_bias(const T *bias, int v) {
    if (!bias) return 0.0f;
    const float b = to_f32(bias[v]), l = b * CE_LOG2E;
    return fabsf(b) < __builtin_inff() ? fminf(fmaxf(l, -3.402823466e38f), 3.402823466e38f) : l;
}

// A row's factor of G: 2^15 g / (largest finite g); below 2^-18 of that one it is 2^13 .. 2^15 in magnitude, with `below` binades (negative) to be
// applied later, so that the row keeps its bits.  An infinity or a NaN is the row's own.
__device__ __forceinline__ float ce_row_factor(float g, float gmax, int &below) {
    if (!(fabsf(g) < __builtin_inff())) return g;
    const float r = g / gmax;
    if (g == 0.0f || fabsf(r) >= 0x1p-18f) return 32768.0f * r;
    int eg, em;
    const float mg = frexpf(g, &eg), mm = frexpf(gmax, &em);      // mg / mm in (1/2, 2)
    below = eg - em + 1;
    return 16384.0f * (mg / mm);
}

// A workgroup keeps its BN hidden rows and walks over a share of the vocabulary's tiles, the next tile's first steps in flight while it
// works on this one's logits (forward pass of 8192 x 16384 x 128 bf16: 81 us, 90 with one tile per workgroup); the running maximum and sum stay
// in each lane until the last tile.
template <typename T, bool SPLIT, bool BACK, int BM, int BN, int WM, int WN, int NST>
__global__ void __launch_bounds__(WM *WN * 64, 2) ce_logits_kernel(CeLogits a, const T *bias) {
    typedef TileGemm<SPLIT, false, false, BM, BN, WM, WN, NST> Gemm;
    constexpr int TM = Gemm::TM, TN = Gemm::TN, NT = WM * WN * 64;
    static_assert(BM <= NT, "one thread per bias entry of a tile");
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    __shared__ __attribute__((aligned(16))) float sb[2][BM];
    int ti, vs;
    const int live = a.sc->live;
    if (!gemm_tile_of(blockIdx.x, ce_padded(live) / BN, a.v_shares, ti, vs)) return;
    const int tv0 = (int)((int64_t)a.tiles_v * vs / a.v_shares), tv1 = (int)((int64_t)a.tiles_v * (vs + 1) / a.v_shares);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int wm = wave / WN, wn = wave % WN;
    // rows or entries on scales of their own, or scales whose product could leave fp32's range: every logit by itself
    const int ex_all = a.sc->ex + a.sc->ew;
    const bool each = (a.sc->x_classes | a.sc->w_classes) != 1 || ex_all > 96 || ex_all < -96;
    const float scale = each ? 1.0f : ldexpf(CE_LOG2E, ex_all);
    // this lane's rows
    uint32_t row[TN];
    int tc[TN];
    float m[TN], s[TN], pf[TN], f[TN];                           // running statistics; backward: top, -, 2^15 r / sum, 2^15 r
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        row[j] = (uint32_t)(ti * BN + wn * TN * 32 + j * 32 + (lane & 31));
        tc[j] = (int)row[j] < live ? a.tc[row[j]] : -1;
        m[j] = CE_NEG_INF;
        s[j] = 0.0f;
        if (BACK) {
            const float2 st = a.stat[row[j]];
            f[j] = tc[j] >= 0 ? 32768.0f : 0.0f;
            if (a.grad) {
                int below = 0;
                if (tc[j] >= 0) f[j] = ce_row_factor(a.grad[a.orig[row[j]]], a.up->gmax, below);
                if (vs == 0 && wm == 0) {
                    const int shift = a.xe[row[j]] - a.sc->ex + below;
                    if (h == 0) a.gs[row[j]] = below;
                    if (h == 0) a.xs[row[j]] = row_scale(shift);
                    if (__any(shift)) ce_add_classes(&a.up->classes, shift ? 1u << row_class(shift) : 0);
                }
            }
            m[j] = st.x;
            pf[j] = st.y * f[j];                                 // f (p - y) = 2^(l - top) (f / sum) - f y
        }
    }
    auto next_bias = [&](int tv) {
        const int v = a.v0 + tv * BM + (int)threadIdx.x;
        return (int)threadIdx.x < BM && v < a.V ? ce_bias(bias, v) : CE_NEG_INF;
    };
    float b_next = next_bias(tv0);
    Gemm g;
    g.init(a.w, a.x, a.v0 + (int64_t)tv0 * BM, 0, 0, (int64_t)ti * BN, 0, 0, lds);
    g.first(0, a.steps);
    for (int tv = tv0; tv < tv1; ++tv) {
        float *tb = sb[tv & 1];
        if ((int)threadIdx.x < BM) tb[threadIdx.x] = b_next;     // read behind the barriers of run(); the other half is still being read
        f32x16 acc[TM][TN];
        float none[TM];
        g.template run<false, false>(0, a.steps, acc, false, none, RowScales{});
        if (tv + 1 < tv1) {
            b_next = next_bias(tv + 1);
            g.a_rows(BM);
            g.first(0, a.steps);
        }
        if (each) {
            int ex[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) ex[j] = a.xe[row[j]];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    __builtin_amdgcn_sched_barrier(0);           // four exponents at a time: all of them spill registers
                    const int4 ew = *(const int4 *)(a.we + a.v0 + tv * BM + wm * TM * 32 + i * 32 + 8 * q + 4 * h);
#pragma unroll
                    for (int j = 0; j < TN; ++j) {
                        acc[i][j][4 * q + 0] = ldexpf(acc[i][j][4 * q + 0] * CE_LOG2E, ex[j] + ew.x);
                        acc[i][j][4 * q + 1] = ldexpf(acc[i][j][4 * q + 1] * CE_LOG2E, ex[j] + ew.y);
                        acc[i][j][4 * q + 2] = ldexpf(acc[i][j][4 * q + 2] * CE_LOG2E, ex[j] + ew.z);
                        acc[i][j][4 * q + 3] = ldexpf(acc[i][j][4 * q + 3] * CE_LOG2E, ex[j] + ew.w);
                    }
                }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 b = *(const float4 *)(tb + wm * TM * 32 + i * 32 + 8 * q + 4 * h);
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    acc[i][j][4 * q + 0] = fmaf(acc[i][j][4 * q + 0], scale, b.x);
                    acc[i][j][4 * q + 1] = fmaf(acc[i][j][4 * q + 1], scale, b.y);
                    acc[i][j][4 * q + 2] = fmaf(acc[i][j][4 * q + 2], scale, b.z);
                    acc[i][j][4 * q + 3] = fmaf(acc[i][j][4 * q + 3], scale, b.w);
                }
            }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            // the target's place in this lane's part of the wave tile: 32 i + 8 q + e
            const int off = tc[j] - (a.v0 + tv * BM) - wm * TM * 32 - 4 * h;
            const bool mine = tc[j] >= 0 && off >= 0 && off < TM * 32 && (off & 4) == 0;
            if (!BACK) {
                float top = m[j];
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = fmaxf(top, acc[i][j][e]);
                const float mm = top == CE_NEG_INF ? 0.0f : top; // nothing but masked entries: a sum of zeros, not of NaN
                s[j] *= __builtin_amdgcn_exp2f(m[j] - mm);
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[j] += __builtin_amdgcn_exp2f(acc[i][j][e] - mm);
                m[j] = top;
                if (__any(mine)) {
                    float l = 0.0f;
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (off == 32 * i + 8 * (e >> 2) + (e & 3)) l = acc[i][j][e];
                    if (mine) a.tlogit[row[j]] = l;
                }
            } else {
                const bool any = __any(mine), edge = (ti + 1) * BN > live;
                // stored order inside 16 columns: 0 1 2 3 8 9 10 11 | 4 5 6 7 12 13 14 15 -- what one lane holds, 16 bytes at a time, at a
                // wave's base and a lane's offset of 32 bits
                half_t *out = a.g + (int64_t)(tv * BM / 32 + wm * TM) * (SPLIT ? 2 : 1) * a.Mp * 32;
                const uint32_t at = row[j] * 32 + h * 8;
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    __builtin_amdgcn_sched_barrier(0);           // one block after the other: all together spill 34 registers (8192 x 16384 x
                                                                 // 128 fp32 backward 493 us against 458)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i][j][e] = __builtin_amdgcn_exp2f(acc[i][j][e] - m[j]) * pf[j];
                    if (edge) {                                  // rows behind the last: 0 times an infinite weight is no number
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[i][j][e] = tc[j] >= 0 ? acc[i][j][e] : 0.0f;
                    }
                    if (any) {
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            acc[i][j][e] -= mine && off == 32 * i + 8 * (e >> 2) + (e & 3) ? f[j] : 0.0f;
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        half8 hi, lo;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float v = acc[i][j][8 * c + e];
                            hi[e] = (half_t)v;
                            if (SPLIT || CE_TWO_PLANES<T, SPLIT>) lo[e] = (half_t)(v - (float)hi[e]);
                        }
                        half_t *o = out + (SPLIT ? (i * 2 + c) * a.Mp * 32 : i * a.Mp * 32 + c * 16) + at;
                        *(half8 *)o = hi;
                        if (SPLIT) *(half8 *)(o + 16) = lo;
                        if (CE_TWO_PLANES<T, SPLIT>) *(half8 *)(o + a.g_plane) = lo;
                    }
                }
            }
        }
    }
    if (!BACK) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const float mo = __shfl_xor(m[j], 32), so = __shfl_xor(s[j], 32), top = fmaxf(m[j], mo), mm = top == CE_NEG_INF ? 0.0f : top;
            const float sum = s[j] * __builtin_amdgcn_exp2f(m[j] - mm) + so * __builtin_amdgcn_exp2f(mo - mm);
            if (h == 0) a.part[(int64_t)(vs * WM + wm) * a.Mp + row[j]] = make_float2(top, sum);
        }
    }
}

// ---- few rows, no gradient: the weight's bytes ------------------------------------------------------------------------------
// Up to 64 rows.  A wave takes 16 vocabulary entries at a time, operands straight from memory into the matrix instruction's
// registers (fp32: v_mfma_f32_16x16x4_f32; lane (r, q) loads the 16 bytes k = 4 q .. of row r, element e feeds the e-th
// instruction for both operands), and keeps the running maximum and sum of every row.  1 x 65536 x 512 bf16 13.5 us: 5.0 TB/s of weight, a
// copy's rate.
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T, bool VEC> struct ScoreLoad;
template <bool VEC> struct ScoreLoad<float, VEC> {
    typedef f32x4 frag;
    static constexpr int KW = 4;
    static __device__ __forceinline__ void mma(const frag &a, const frag &b, f32x4 &c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    }
};
template <bool VEC> struct ScoreLoad<half_t, VEC> {
    typedef half8 frag;
    static constexpr int KW = 8;
    static __device__ __forceinline__ void mma(const frag &a, const frag &b, f32x4 &c) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <bool VEC> struct ScoreLoad<bf16_t, VEC> {
    typedef bf8 frag;
    static constexpr int KW = 8;
    static __device__ __forceinline__ void mma(const frag &a, const frag &b, f32x4 &c) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

template <typename T, bool VEC>
__device__ __forceinline__ typename ScoreLoad<T, VEC>::frag score_load(const T *row, int k, int D) {
    typedef ScoreLoad<T, VEC> L;
    Pack<T, L::KW> p;
    if (VEC) {
        if (k < D) return __builtin_bit_cast(typename L::frag, *(const Pack<T, L::KW> *)(row + k));
#pragma unroll
        for (int e = 0; e < L::KW; ++e) p.v[e] = from_f32<T>(0.0f);
    } else {
#pragma unroll
        for (int e = 0; e < L::KW; ++e) p.v[e] = k + e < D ? row[k + e] : from_f32<T>(0.0f);
    }
    return __builtin_bit_cast(typename L::frag, p);
}

// G groups of 16 entries at a time: the hidden states' operands, read from the caches, serve all of them.
template <typename T, bool VEC, int NT, int G>
__global__ void __launch_bounds__(256) ce_score_kernel(const T *x, int64_t ldx, int M, const T *w, int64_t ldw, int V, int D, const T *bias,
                                                       const int64_t *target, float2 *part, float *tlogit, CeScalars *sc) {
    typedef ScoreLoad<T, VEC> L;
    constexpr int KS = 4 * L::KW, U = NT == 1 && G == 1 ? 4 : 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    if (blockIdx.x == 0 && threadIdx.x == 0) sc->ticket = 0;
    const T *xr[NT];
    float m[NT], s[NT];
    int64_t t[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int i = n * 16 + r < M ? n * 16 + r : M - 1;
        xr[n] = x + i * ldx;
        t[n] = n * 16 + r < M ? target[i] : -1;
        m[n] = CE_NEG_INF;
        s[n] = 0.0f;
    }
    const int groups = (V + 15) / 16;
    for (int g0 = (blockIdx.x * 4 + wave) * G; g0 < groups; g0 += gridDim.x * 4 * G) {
        const T *wr[G];
        f32x4 acc[G][NT];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int v = (g0 + g) * 16 + r;
            wr[g] = w + (int64_t)(v < V ? v : V - 1) * ldw;
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[g][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (int k = q * L::KW; k < D + q * L::KW; k += U * KS) {
            typename L::frag fw[G][U], fx[NT][U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int g = 0; g < G; ++g) fw[g][u] = score_load<T, VEC>(wr[g], k + u * KS, D);
#pragma unroll
                for (int n = 0; n < NT; ++n) fx[n][u] = score_load<T, VEC>(xr[n], k + u * KS, D);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int n = 0; n < NT; ++n) L::mma(fw[g][u], fx[n][u], acc[g][n]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float l[G][4], top = m[n];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int v = (g0 + g) * 16 + 4 * q + e;
                    l[g][e] = v < V ? fmaf(acc[g][n][e], CE_LOG2E, ce_bias(bias, v)) : CE_NEG_INF;
                    top = fmaxf(top, l[g][e]);
                    if (t[n] == v) tlogit[n * 16 + r] = l[g][e];
                }
            const float mm = top == CE_NEG_INF ? 0.0f : top;
            s[n] *= __builtin_amdgcn_exp2f(m[n] - mm);
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n] += __builtin_amdgcn_exp2f(l[g][e] - mm);
            m[n] = top;
        }
    }
    __shared__ float2 red[4][NT * 16];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        for (int o = 16; o < 64; o <<= 1) {
            const float mo = __shfl_xor(m[n], o), so = __shfl_xor(s[n], o), top = fmaxf(m[n], mo), mm = top == CE_NEG_INF ? 0.0f : top;
            s[n] = s[n] * __builtin_amdgcn_exp2f(m[n] - mm) + so * __builtin_amdgcn_exp2f(mo - mm);
            m[n] = top;
        }
        if (q == 0) red[wave][n * 16 + r] = make_float2(m[n], s[n]);
    }
    __syncthreads();
    if ((int)threadIdx.x < NT * 16) {
        float top = CE_NEG_INF, sum = 0.0f;
        for (int k = 0; k < 4; ++k) top = fmaxf(top, red[k][threadIdx.x].x);
        const float mm = top == CE_NEG_INF ? 0.0f : top;
        for (int k = 0; k < 4; ++k) sum += red[k][threadIdx.x].y * __builtin_amdgcn_exp2f(red[k][threadIdx.x].x - mm);
        part[(int64_t)blockIdx.x * CE_SCORE_ROWS + threadIdx.x] = make_float2(top, sum);
    }
}

// ---- rows: join the tiles' statistics, losses, their sum --------------------------------------------------------------------
// 2^rsh rows per workgroup, 256 >> rsh threads stride over one row's parts.  The last workgroup to finish adds the workgroups'
// sums in their order, in fp64.  PACKED: rows are those that are there (orig, tc), else the caller's own (few rows, ce_score_kernel).
struct CeRows {
    const float2 *part;
    int64_t ldp;
    int parts;
    const float *tlogit;
    const int64_t *target;
    const int32_t *tc, *orig;
    int64_t M;
    int V, rsh, reduction;
    float2 *stat;
    float *loss;
    double2 *sums;
    CeScalars *sc;
};
template <bool PACKED> __global__ void __launch_bounds__(256) ce_rows_kernel(CeRows a) {
    __shared__ float2 sh[256];
    __shared__ double2 tot[256];
    __shared__ bool last;
    const int rows = 1 << a.rsh, segs = 256 >> a.rsh, r = threadIdx.x & (rows - 1), seg = threadIdx.x >> a.rsh;
    const int64_t i = (int64_t)blockIdx.x * rows + r, n = PACKED ? a.sc->live : a.M;
    float m = CE_NEG_INF, s = 0.0f;
    if (i < n) {
        constexpr int U = 4;
        for (int p = seg; p < a.parts; p += segs * U) {
            float2 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = a.part[(int64_t)(p + u * segs < a.parts ? p + u * segs : p) * a.ldp + i];
            float top = m;
#pragma unroll
            for (int u = 0; u < U; ++u) top = fmaxf(top, v[u].x);
            const float mm = top == CE_NEG_INF ? 0.0f : top;
            s *= __builtin_amdgcn_exp2f(m - mm);
#pragma unroll
            for (int u = 0; u < U; ++u) s += p + u * segs < a.parts ? v[u].y * __builtin_amdgcn_exp2f(v[u].x - mm) : 0.0f;
            m = top;
        }
    }
    sh[threadIdx.x] = make_float2(m, s);
    __syncthreads();
    double2 mine = make_double2(0.0, 0.0);
    if (seg == 0) {
        const int64_t t = i < n ? (PACKED ? (int64_t)a.tc[i] : a.target[i]) : -1;
        float2 stat = make_float2(__builtin_inff(), 0.0f);
        float l = 0.0f;
        if (t >= 0) {
            float top = CE_NEG_INF, sum = 0.0f;
            for (int k = 0; k < segs; ++k) top = fmaxf(top, sh[(k << a.rsh) + r].x);
            const float mm = top == CE_NEG_INF ? 0.0f : top;
            for (int k = 0; k < segs; ++k) sum += sh[(k << a.rsh) + r].y * __builtin_amdgcn_exp2f(sh[(k << a.rsh) + r].x - mm);
            const float ls = log2f(sum);
            // kept apart: the backward pass forms 2^(l - top) / sum, which keeps its precision however large the logits are
            stat = make_float2(top, t < a.V ? 1.0f / sum : __builtin_nanf(""));
            // (top - target's logit) first: the two are near each other where the loss is small
            l = t < a.V ? (float)(((double)(top - a.tlogit[i]) + (double)ls) * CE_LN2) : __builtin_nanf("");
            mine = make_double2((double)l, 1.0);
        }
        if (PACKED && a.stat && i < ce_padded((int)n)) a.stat[i] = stat;
        if (a.reduction == 0) {
            if (!PACKED && i < a.M) a.loss[i] = l;
            if (PACKED && i < n) a.loss[a.orig[i]] = l;
            if (PACKED && i < a.M && a.target[i] < 0) a.loss[i] = 0.0f;
        }
    }
    if (a.reduction == 0) return;
    tot[threadIdx.x] = mine;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if ((int)threadIdx.x < o) { tot[threadIdx.x].x += tot[threadIdx.x + o].x; tot[threadIdx.x].y += tot[threadIdx.x + o].y; }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        // written through to where every XCD reads it, and there before the ticket is drawn: no cache has to be flushed
        __hip_atomic_store(&a.sums[blockIdx.x].x, tot[0].x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&a.sums[blockIdx.x].y, tot[0].y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        last = __hip_atomic_fetch_add(&a.sc->ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    mine = make_double2(0.0, 0.0);
    for (unsigned k = threadIdx.x; k < gridDim.x; k += 256) {
        mine.x += __hip_atomic_load(&a.sums[k].x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        mine.y += __hip_atomic_load(&a.sums[k].y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    tot[threadIdx.x] = mine;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if ((int)threadIdx.x < o) { tot[threadIdx.x].x += tot[threadIdx.x + o].x; tot[threadIdx.x].y += tot[threadIdx.x + o].y; }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double c = tot[0].y;
        a.loss[0] = (float)(a.reduction == 1 ? (c > 0.0 ? tot[0].x / c : 0.0) : tot[0].x);
    }
}

// largest finite |grad| over the rows that are there (reduction none); a row whose gradient is no number keeps that to itself
__global__ void __launch_bounds__(1024) ce_gmax_kernel(const float *grad, const int64_t *target, int64_t M, CeUpstream *up) {
    __shared__ float sh[16];
    float a = 0.0f;
    for (int64_t i = threadIdx.x; i < M; i += 1024)
        if (target[i] >= 0) {
            const float g = fabsf(grad[i]);
            a = g < __builtin_inff() ? fmaxf(a, g) : a;
        }
    for (int o = 32; o; o >>= 1) a = fmaxf(a, __shfl_xor(a, o));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 16; ++k) a = fmaxf(a, sh[k]);
        up->gmax = a > 0.0f ? a : 1.0f;
        up->classes = 1;
    }
}

// ---- gradient products ------------------------------------------------------------------------------------------------------
// what takes a sum over G back to the gradient: 2^-15 times the other operand's scale, a power of two, and then max g (in one factor a
// small max g would lose bits below the smallest normal number)
struct CeFactor { float two, g; };
__device__ __forceinline__ CeFactor ce_unscale(const CeScalars *sc, const float *grad, const CeUpstream *up, int reduction, int e) {
    const float g = reduction == 0 ? up->gmax : reduction == 1 ? grad[0] / (float)(sc->live > 0 ? sc->live : 1) : grad[0];
    return CeFactor{ldexpf(1.0f, e - 15), g};
}

struct CeGrad {
    GemmOperand g, o;         // G and the other operand (weight or hidden states)
    int64_t rows, out0;       // dweight: output rows of this call, the first one's index in the output
    int tiles_d, steps, splits, blocks;
    int64_t ok0;              // first row of the other operand
    const int32_t *o_scales;  // its rows' words (vocab_gemm.h), from there
    int g_panels, o_panels;
    void *out;                // final output (nothing to add up), [..][D]
    float *part;              // [splits][part_rows][D] sums, or NULL
    int64_t part_rows;
    int add;                  // part += (later pieces of the vocabulary)
};
struct CeGrads {
    CeGrad x, w;              // dhidden, dweight
    const CeScalars *sc;
    const float *grad;
    const CeUpstream *up;     // reduction none, as in CeLogits; gs else NULL
    const int32_t *gs;
    const int64_t *target;
    const int32_t *orig;      // dhidden: the caller's row of a row that is there
    int64_t M, g_plane;
    int reduction, D, zero_blocks;
    float *part_b;            // dbias: [w.splits][ldb] sums in G's stored column order, or NULL
    int64_t ldb;
};

template <int TM, int TN> __device__ __forceinline__ void ce_rescale(f32x16 (&acc)[TM][TN], int by) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = ldexpf(acc[i][j][e], by);
}

// WEIGHT: dweight (G read transposed, output rows = vocabulary entries in G's stored column order), else dhidden
template <typename T, bool SPLIT, bool WEIGHT, int BM, int BN, int WM, int WN, int NST>
__device__ __forceinline__ void ce_grad_tile(const CeGrads &a, const CeGrad &c, int bid, char *lds) {
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int PC = SPLIT ? 16 : 32;                        // columns per panel
    int tr, td;
    const int live = a.sc->live;
    const int64_t rows = WEIGHT ? c.rows : live;
    const int tiles_r = (int)((rows + BM - 1) / BM), per = (tiles_r * c.tiles_d + 7) / 8 * 8, z = per ? bid / per : c.splits;
    if (z >= c.splits || !gemm_tile_of(bid - z * per, tiles_r, c.tiles_d, tr, td)) return;
    const int64_t r0 = (int64_t)tr * BM;
    const int d0 = td * BN;
    const int64_t plane_steps = WEIGHT ? ce_padded(live) / PC : c.steps, steps = plane_steps * (CE_TWO_PLANES<T, SPLIT> ? 2 : 1);
    const int s0 = (int)(steps * z / c.splits), s1 = (int)(steps * (z + 1) / c.splits);
    f32x16 acc[TM][TN];
    const int gp = WEIGHT ? (int)(r0 / PC) : 0, op = d0 / PC;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int wm = wave / WN, wn = wave % WN;
    // dbias: the sums over k of G^T, which the first column of waves of the first column of tiles has in registers anyway
    const bool sums = WEIGHT && a.part_b && td == 0 && wn == 0;
    float asum[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) asum[i] = 0.0f;
    TileGemm<SPLIT, WEIGHT, true, BM, BN, WM, WN, NST> g;
    g.init(c.g, c.o, WEIGHT ? 0 : r0, gp, c.g_panels - gp, c.ok0, op, c.o_panels - op, lds);
    if (CE_TWO_PLANES<T, SPLIT>) g.two_planes(a.g_plane, (int)plane_steps);
    const uint32_t classes = !WEIGHT ? a.sc->w_classes : a.gs ? a.up->classes : a.sc->x_classes;
    if (classes == 1) {
        g.first(s0, s1);
        g.template run<WEIGHT, false>(s0, s1, acc, sums, asum, RowScales{});
    } else {
        int at = 0;                                            // the class on whose scale acc is
        decltype(g)::clear(acc);
        for (int k = ROW_CLASSES - 1; k >= 0; --k) {
            if (!(classes >> k & 1)) continue;
            const RowScales rs{c.o_scales, WEIGHT ? a.gs : nullptr, k};
            int c0 = s0, c1 = s1;
            class_steps<PC>(rs, CE_TWO_PLANES<T, SPLIT> ? (int)plane_steps : INT32_MAX, c0, c1, lane);
            if (c0 == c1) continue;
            if (at) ce_rescale(acc, 16 * (k - at));
            at = k;
            g.first(c0, c1);
            g.template run<WEIGHT, true>(c0, c1, acc, sums, asum, rs);
        }
        if (at) ce_rescale(acc, -16 * at);
    }
    if (sums) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const float t = asum[i] + __shfl_xor(asum[i], 32);
            if (h == 0) a.part_b[z * a.ldb + r0 + wm * TM * 32 + i * 32 + lane] = t;
        }
    }
    if (!c.out) return;                                        // only dbias is asked for
    const CeFactor f = ce_unscale(a.sc, a.grad, a.up, a.reduction, WEIGHT ? a.sc->ex : a.sc->ew);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int pos = (e & 3) + 8 * (e >> 2) + 4 * h;
            const int loc = WEIGHT ? (pos & ~12) | ((pos & 4) << 1) | ((pos & 8) >> 1) : pos;
            const int64_t row = r0 + wm * TM * 32 + i * 32 + loc;
            if (row >= rows) continue;
            const int64_t to = WEIGHT ? c.out0 + row : c.part ? 0 : a.orig[row];
            const int below = !WEIGHT && a.gs ? a.gs[row] : 0;
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int d = d0 + wn * TN * 32 + j * 32 + (lane & 31);
                if (d >= a.D) continue;
                const float v = acc[i][j][e];
                if (c.part) {
                    float *p = c.part + ((int64_t)z * c.part_rows + row) * a.D + d;
                    *p = c.add ? *p + v : v;
                } else {
                    ((T *)c.out)[to * a.D + d] = from_f32<T>(ldexpf(v * f.two * f.g, below));
                }
            }
        }
}

// Both gradient products in one launch: they read the same G, and the workgroups of one fill what the other's leave idle.  The last
// workgroups zero dhidden of the absent rows.  16384 x 65536 x 1024 bf16 2 x 2.02 ms: 1.09 PFLOP/s (library products of these sizes 1.14 and
// 1.51); 4096 x 16384 x 512 fp32 355 us: 387 TFLOP/s; 19700 x 1024 x 128 fp32 51 us: 203; 1237 x 5003 x 201 fp16, two planes of G, 48 us (one: 23).
// The matrix pipe is busy for 58 % (bf16) and 67 % (fp32) of the cycles, at 1.9 GHz, 34 % in the third case, whose tiles have few steps.
template <typename T, bool SPLIT, int BM, int BN, int WM, int WN, int NST>
__global__ void __launch_bounds__(WM *WN * 64, 2) ce_grads_kernel(CeGrads a) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int bid = blockIdx.x;
    if (bid < a.x.blocks) ce_grad_tile<T, SPLIT, false, BM, BN, WM, WN, NST>(a, a.x, bid, lds);
    else if (bid < a.x.blocks + a.w.blocks) ce_grad_tile<T, SPLIT, true, BM, BN, WM, WN, NST>(a, a.w, bid - a.x.blocks, lds);
    else {                                                     // dhidden of the absent rows
        const int wave = (bid - a.x.blocks - a.w.blocks) * (WM * WN) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
        for (int64_t r = wave; r < a.M; r += (int64_t)a.zero_blocks * WM * WN)
            if (a.target[r] < 0)
                for (int d = lane; d < a.D; d += 64) ((T *)a.x.out)[r * a.D + d] = from_f32<T>(0.0f);
    }
}

// out[r][d] = factor * sum over splits of part[s][r][d], the splits in their order; VE elements per thread and trip
template <typename T, int VE>
__device__ __forceinline__ void ce_join(const CeGrads &a, const CeGrad &c, bool weight, int bid, int blocks) {
    const int64_t n = (weight ? c.rows : (int64_t)a.sc->live) * a.D, stride = c.part_rows * a.D;
    const CeFactor f = ce_unscale(a.sc, a.grad, a.up, a.reduction, weight ? a.sc->ex : a.sc->ew);
    for (int64_t k = ((int64_t)bid * 256 + threadIdx.x) * VE; k < n; k += (int64_t)blocks * 256 * VE) {
        const int64_t row = k / a.D;
        float v[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = 0.0f;
        constexpr int U = 8;
        for (int s = 0; s < c.splits; s += U) {
            Pack<float, VE> p[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                p[u] = *(const Pack<float, VE> *)(c.part + (s + u < c.splits ? s + u : s) * stride + k);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s + u < c.splits)
#pragma unroll
                    for (int e = 0; e < VE; ++e) v[e] += p[u].v[e];
        }
        const int below = !weight && a.gs ? a.gs[row] : 0;
        T *out = (T *)c.out + (weight ? c.out0 + row : (int64_t)a.orig[row]) * a.D + (k - row * a.D);
#pragma unroll
        for (int e = 0; e < VE; ++e) out[e] = from_f32<T>(ldexpf(v[e] * f.two * f.g, below));
    }
}

// what is left of a piece in one launch: dhidden and dweight from their partial sums (bx / bw workgroups), dbias
template <typename T, int VE>
__global__ void __launch_bounds__(256) ce_join_kernel(CeGrads a, int bx, int bw, int live, T *dbias) {
    const int bid = blockIdx.x;
    if (bid < bx) { ce_join<T, VE>(a, a.x, false, bid, bx); return; }
    if (bid < bx + bw) { ce_join<T, VE>(a, a.w, true, bid - bx, bw); return; }
    const int v = (bid - bx - bw) * 256 + threadIdx.x;
    if (v >= live) return;
    const int pos = (v & ~12) | ((v & 4) << 1) | ((v & 8) >> 1);
    float s = 0.0f;
    for (int k = 0; k < a.w.splits; ++k) s += a.part_b[k * a.ldb + pos];
    const CeFactor f = ce_unscale(a.sc, a.grad, a.up, a.reduction, 0);
    dbias[v] = from_f32<T>(s * f.two * f.g);
}

// ---- host -------------------------------------------------------------------------------------------------------------------
static inline size_t ce_up(size_t n) { return (n + 255) & ~(size_t)255; }
static inline int64_t ce_pad(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

static CeShape ce_shape(const tnp_vocab_ce *p) {
    CeShape s;
    s.M = p->M; s.Mp = ce_pad(p->M, CE_ROW_PAD);
    s.V = p->V; s.Vp = (int)ce_pad(p->V, CE_COL_PAD); s.D = p->D;
    s.split = p->dtype == TNP_F32;
    s.panels = s.split ? (p->D + 15) / 16 : (p->D + 31) / 32;
    return s;
}

struct CeSaved { CeScalars *sc; float2 *stat; int32_t *tc, *orig, *xe, *xs, *we, *ws; half_t *x, *w; size_t bytes; };
static CeSaved ce_saved(const CeShape &s, void *base) {
    CeSaved v;
    char *p = (char *)base;
    v.sc = (CeScalars *)p; p += 256;
    v.stat = (float2 *)p; p += s.Mp * 8;               // Mp and Vp are multiples of 256: every part stays aligned
    v.tc = (int32_t *)p; p += s.Mp * 4;
    v.orig = (int32_t *)p; p += s.Mp * 4;
    v.xe = (int32_t *)p; p += s.Mp * 4;
    v.xs = (int32_t *)p; p += s.Mp * 4;
    v.we = (int32_t *)p; p += (size_t)s.Vp * 4;
    v.ws = (int32_t *)p; p += (size_t)s.Vp * 4;
    v.x = (half_t *)p; p += (size_t)s.Mp * s.panels * 64;
    v.w = (half_t *)p; p += (size_t)s.Vp * s.panels * 64;
    v.bytes = (size_t)(p - (char *)base);
    return v;
}

static bool ce_scores(const tnp_vocab_ce *p) { return !p->saved && p->M <= CE_SCORE_ROWS; }
static int ce_score_groups(const tnp_vocab_ce *p) { return p->M > 16 && p->V >= CE_SCORE_GROUPS_FROM ? CE_SCORE_GROUPS : 1; }
static int ce_score_blocks(const tnp_vocab_ce *p) {
    const int each = 64 * ce_score_groups(p), g = (p->V + each - 1) / each;
    return g < 1024 ? g : 1024;
}
// rows per workgroup of the join: few rows share the threads, many rows with few parts keep the workgroups few (each draws a ticket:
// 24576 rows of 16 parts 14 us at 32 rows, 7 at 128; 16384 rows of 512 parts 20 us at 32 rows, 37 at 128)
static int ce_rows_shift(int64_t M, int parts) { return M <= CE_SCORE_ROWS ? 2 : M >= 8192 && parts <= 32 ? 7 : 5; }

// shares of the hidden states' rows: at least eight rows each
static int ce_x_blocks(int64_t M) { return (int)((M + 7) / 8 < CE_AMAX_BLOCKS ? (M + 7) / 8 : CE_AMAX_BLOCKS); }

// Shares that the `tiles_v` vocabulary tiles are split into for each of `tiles_i` row tiles, `slots` workgroups running at a time: the
// fewest rounds of workgroups times tiles per workgroup, and of those the fewest shares.  No bound on the shares: 200 x 65536 x 512 bf16 forward
// 72 us, 97 with at most 64 of them.
static int ce_shares(int64_t tiles_i, int tiles_v, int slots) {
    int best = 1;
    int64_t cost = INT64_MAX;
    for (int n = 1; n <= tiles_v; ++n) {
        const int64_t rounds = (tiles_i * n + slots - 1) / slots, c = rounds * ((tiles_v + n - 1) / n);
        if (c < cost) { cost = c; best = n; }
        if (tiles_i * n >= 2 * slots) break;
    }
    return best;
}
// 256 x 256 tiles of logits (eight waves) from two rounds of workgroups and eight steps on: 4096 x 16384 x 1024 fp32 forward 381 us
// against 437, 8192 x 16384 x 128 bf16 (four steps) 95 against 86
static bool ce_big(const CeShape &s) { return (s.Mp / 256) * (int64_t)(s.Vp / 256) >= 512 && s.panels >= 8; }
// slots: one workgroup of the 256 tiles per CU, three of the 128 ones
static int ce_logit_shares(const CeShape &s, int64_t cols) {
    return ce_big(s) ? ce_shares(s.Mp / 256, (int)(cols / 256), 256) : ce_shares(s.Mp / 128, (int)(cols / 128), 768);
}

struct CeForward { CeSaved saved; float *amax; int *count; float2 *part; float *tlogit; double2 *sums; int parts; size_t bytes; };
static CeForward ce_forward_layout(const tnp_vocab_ce *p, void *ws) {
    CeForward f;
    const CeShape s = ce_shape(p);
    char *w = (char *)ws;
    f.parts = ce_scores(p) ? ce_score_blocks(p) : 2 * ce_logit_shares(s, s.Vp);
    const int64_t rows = ce_scores(p) ? CE_SCORE_ROWS : s.Mp;
    f.amax = (float *)w; w += ce_up(2 * CE_AMAX_BLOCKS * 4);
    f.count = (int *)w; w += ce_up(CE_AMAX_BLOCKS * 4);
    f.part = (float2 *)w; w += ce_up((size_t)f.parts * rows * 8);
    f.tlogit = (float *)w; w += ce_up(rows * 4);
    f.sums = (double2 *)w; w += ce_up((size_t)((s.Mp >> ce_rows_shift(p->M, f.parts)) + 1) * 16);
    f.saved = ce_saved(s, p->saved ? p->saved : w);
    if (!p->saved) w += ce_scores(p) ? 256 : f.saved.bytes;
    f.bytes = (size_t)(w - (char *)ws);
    return f;
}

// columns of G that are formed at a time, and the tiles and splits of the two gradient products
struct CeBackward {
    int piece, pieces;
    int64_t ldg;
    half_t *g;
    int tile, splits_x, splits_w;
    CeUpstream *up;
    int32_t *gs, *xs;
    float *part_x, *part_w, *part_b;
    size_t bytes;
};
// G of a piece of the vocabulary: at most this much or 256 entries of all rows, whichever is more (rows are not split: 2^23 of them are 4 GB in
// bf16, 8 GB in two fp16 numbers)
static constexpr size_t CE_PIECE_BYTES = (size_t)1 << 30;      // of 288 GB; 16384 x 65536 x 1024 bf16 backward 7.59 ms with 256 MB, 6.42 with 512, 6.32, 6.27 with 2 GB

static CeBackward ce_backward_layout(const tnp_vocab_ce *p, void *ws) {
    CeBackward b;
    const CeShape s = ce_shape(p);
    const int planes = ce_g_planes(p->dtype), ks = s.split ? 16 : 32, runs = s.split ? 1 : planes;     // runs of the products over G
    int64_t most = (int64_t)(CE_PIECE_BYTES / ((size_t)s.Mp * 2 * planes)) / 256 * 256;
    if (most < 256) most = 256;
    b.pieces = (int)((s.Vp + most - 1) / most);
    b.piece = (int)ce_pad((s.Vp + b.pieces - 1) / b.pieces, 256);
    b.pieces = (s.Vp + b.piece - 1) / b.piece;
    b.ldg = (int64_t)b.piece * planes;
    // 256 x 256 tiles (eight waves) where they are many steps' work: 16384 x 4096 x 512 bf16 backward 248 us against 285, 8192 x 16384 x
    // 128 (65536 tile steps) 229 against 218
    const int64_t td = (p->D + 127) / 128, small_x = s.Mp / 128 * td, small_w = b.piece / 128 * td;
    const int sx = b.piece / ks * runs, sw = (int)(s.Mp / ks) * runs;
    b.tile = small_x * sx + small_w * sw >= 131072 && p->D > 128 ? 256 : 128;
    // both products share a launch: every workgroup gets about the same number of steps, at least 8
    const int64_t tx = s.Mp / b.tile * ((p->D + b.tile - 1) / b.tile), tw = b.piece / b.tile * ((p->D + b.tile - 1) / b.tile);
    int64_t each = (tx * sx + tw * sw) / (b.tile == 256 ? 256 : 512);
    if (each < 16) each = 16;
    const int64_t nx = (sx + each / 2) / each, nw = (sw + each / 2) / each;
    b.splits_x = (int)(nx < 1 ? 1 : nx);
    b.splits_w = (int)(nw < 1 ? 1 : nw);
    char *w = (char *)ws;
    b.up = (CeUpstream *)w; w += 256;
    b.gs = p->reduction == 0 ? (int32_t *)w : nullptr;
    b.xs = b.gs ? b.gs + s.Mp : nullptr;
    if (b.gs) w += ce_up((size_t)s.Mp * 8);
    b.g = (half_t *)w; w += ce_up((size_t)s.Mp * b.ldg * 2);
    b.part_x = b.splits_x > 1 || b.pieces > 1 ? (float *)w : nullptr;
    if (b.part_x) w += ce_up((size_t)b.splits_x * s.Mp * p->D * 4);
    b.part_w = b.splits_w > 1 ? (float *)w : nullptr;
    if (b.part_w) w += ce_up((size_t)b.splits_w * b.piece * p->D * 4);
    b.part_b = p->bias ? (float *)w : nullptr;
    if (b.part_b) w += ce_up((size_t)b.splits_w * b.piece * 4);
    b.bytes = (size_t)(w - (char *)ws);
    return b;
}

static int ce_check(const tnp_vocab_ce *p, const char *who) {
    if (!p) TNP_FAIL(-1, "%s: NULL arguments", who);
    if (!dtype_known(p->dtype)) TNP_FAIL(-1, "%s: unknown dtype %d", who, p->dtype);
    if (p->reduction < 0 || p->reduction > 2) TNP_FAIL(-1, "%s: unknown reduction %d", who, p->reduction);
    if (p->M < 0 || p->M > (1 << 23)) TNP_FAIL(-1, "%s: %lld rows (0 .. 2^23)", who, (long long)p->M);
    if (p->V < 1 || p->V > (1 << 23)) TNP_FAIL(-1, "%s: vocabulary of %d (1 .. 2^23)", who, p->V);
    if (p->D < 1 || p->D > 16384) TNP_FAIL(-1, "%s: %d columns (1 .. 16384)", who, p->D);
    if (p->ld_hidden < p->D || p->ld_weight < p->D) TNP_FAIL(-1, "%s: a row stride is smaller than the %d columns", who, p->D);
    return 0;
}

static int ce_vec(int dtype, int D, int64_t ld, const void *p) {       // elements per load of a row: 16 bytes or one
    const int ve = 16 / (int)dtype_bytes(dtype);
    return D % ve == 0 && ld % ve == 0 && (uintptr_t)p % 16 == 0 ? ve : 1;
}

template <typename KernT>
static int ce_lds(KernT kern, size_t smem, size_t *done) {             // done: per device
    int dev = 0;
    TNP_HIP(hipGetDevice(&dev));
    if (dev < VOCAB_MAX_DEVICES && done[dev] >= smem) return 0;
    TNP_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (dev < VOCAB_MAX_DEVICES) done[dev] = smem;
    return 0;
}

template <typename T, bool SPLIT, bool BACK, int BM, int BN, int WM, int WN, int NST>
static int ce_launch_logits(CeLogits a, int64_t cols, const T *bias, hipStream_t s) {
    a.tiles_v = (int)(cols / BM);
    const size_t smem = NST * (BM + BN) * 64;
    static size_t done[VOCAB_MAX_DEVICES] = {0};
    auto kern = ce_logits_kernel<T, SPLIT, BACK, BM, BN, WM, WN, NST>;
    if (int rc = ce_lds(kern, smem, done)) return rc;
    hipLaunchKernelGGL(kern, dim3(gemm_grid(a.Mp / BN * a.v_shares)), dim3(WM * WN * 64), smem, s, a, bias);
    TNP_HIP(hipGetLastError());
    return 0;
}
template <typename T, bool SPLIT, bool BACK>
static int ce_logits(const CeLogits &a, int64_t cols, bool big, const T *bias, hipStream_t s) {
    return big ? ce_launch_logits<T, SPLIT, BACK, 256, 256, 2, 4, 4>(a, cols, bias, s) : ce_launch_logits<T, SPLIT, BACK, 128, 128, 2, 2, 3>(a, cols, bias, s);
}

template <typename T, bool SPLIT, int BM, int BN, int WM, int WN, int NST>
static int ce_launch_grads(CeGrads &a, hipStream_t s) {
    const size_t smem = NST * (BM + BN) * 64;
    static size_t done[VOCAB_MAX_DEVICES] = {0};
    auto kern = ce_grads_kernel<T, SPLIT, BM, BN, WM, WN, NST>;
    if (int rc = ce_lds(kern, smem, done)) return rc;
    for (CeGrad *c : {&a.x, &a.w}) {
        const int64_t tiles_r = ((c == &a.w ? c->rows : a.M) + BM - 1) / BM;
        c->tiles_d = c->out ? (a.D + BN - 1) / BN : 1;
        c->blocks = c->out || (c == &a.w && a.part_b) ? gemm_grid(tiles_r * c->tiles_d) * c->splits : 0;
    }
    const int blocks = a.x.blocks + a.w.blocks + a.zero_blocks;
    if (blocks) {
        hipLaunchKernelGGL(kern, dim3(blocks), dim3(WM * WN * 64), smem, s, a);
        TNP_HIP(hipGetLastError());
    }
    return 0;
}

template <typename T, bool VEC, int NT, int G>
static int ce_score_run(const tnp_vocab_ce *p, const CeForward &f, hipStream_t s) {
    hipLaunchKernelGGL((ce_score_kernel<T, VEC, NT, G>), dim3(ce_score_blocks(p)), dim3(256), 0, s, (const T *)p->hidden, p->ld_hidden, (int)p->M,
                       (const T *)p->weight, p->ld_weight, p->V, p->D, (const T *)p->bias, p->target, f.part, f.tlogit, f.saved.sc);
    TNP_HIP(hipGetLastError());
    return 0;
}
template <typename T, bool VEC>
static int ce_score(const tnp_vocab_ce *p, const CeForward &f, hipStream_t s) {
    const bool one = ce_score_groups(p) == 1;
    switch ((p->M + 15) / 16) {
        case 1: return ce_score_run<T, VEC, 1, 1>(p, f, s);
        case 2: return one ? ce_score_run<T, VEC, 2, 1>(p, f, s) : ce_score_run<T, VEC, 2, CE_SCORE_GROUPS>(p, f, s);
        case 3: return one ? ce_score_run<T, VEC, 3, 1>(p, f, s) : ce_score_run<T, VEC, 3, CE_SCORE_GROUPS>(p, f, s);
        default: return one ? ce_score_run<T, VEC, 4, 1>(p, f, s) : ce_score_run<T, VEC, 4, CE_SCORE_GROUPS>(p, f, s);
    }
}

template <typename T, int VX, int VW, bool SPLIT>
static int ce_pack(const tnp_vocab_ce *p, const CeShape &sh, const CeForward &f, hipStream_t s) {
    hipLaunchKernelGGL((ce_amax_kernel<T, VX, VW>), dim3(2 * CE_AMAX_BLOCKS), dim3(256), 0, s, (const T *)p->hidden,
                       p->ld_hidden, p->M, p->target, (const T *)p->weight, p->ld_weight, p->V, p->D, ce_x_blocks(p->M), f.amax, f.count, f.saved.sc);
    TNP_HIP(hipGetLastError());
    const int xb = ce_x_blocks(p->M), wb = sh.Vp / 64 < 2048 ? sh.Vp / 64 : 2048;
    hipLaunchKernelGGL((ce_pack_kernel<T, VX, VW, SPLIT>), dim3(xb + wb), dim3(256), 0, s, (const T *)p->hidden, p->ld_hidden, p->target,
                       (const T *)p->weight, p->ld_weight, sh, f.amax, f.count, f.saved.sc, f.saved.x, f.saved.w,
                       f.saved.orig, f.saved.tc, f.saved.xe, f.saved.xs, f.saved.we, f.saved.ws, xb);
    TNP_HIP(hipGetLastError());
    return 0;
}

template <typename T, int VE, bool SPLIT>
static int ce_forward(const tnp_vocab_ce *p, const CeForward &f, float *loss, hipStream_t s) {
    const CeShape sh = ce_shape(p);
    const bool vx = ce_vec(p->dtype, p->D, p->ld_hidden, p->hidden) > 1, vw = ce_vec(p->dtype, p->D, p->ld_weight, p->weight) > 1;
    int rc;
    if (ce_scores(p)) {
        rc = vx && vw ? ce_score<T, true>(p, f, s) : ce_score<T, false>(p, f, s);
        if (rc) return rc;
    } else {
        rc = vx && vw ? ce_pack<T, VE, VE, SPLIT>(p, sh, f, s) : vw ? ce_pack<T, 1, VE, SPLIT>(p, sh, f, s)
             : vx ? ce_pack<T, VE, 1, SPLIT>(p, sh, f, s) : ce_pack<T, 1, 1, SPLIT>(p, sh, f, s);
        if (rc) return rc;
        CeLogits a = {};
        a.w = GemmOperand{f.saved.w, sh.Vp, 0};
        a.x = GemmOperand{f.saved.x, sh.Mp, 0};
        a.sc = f.saved.sc; a.tc = f.saved.tc; a.orig = f.saved.orig; a.xe = f.saved.xe; a.we = f.saved.we; a.Mp = sh.Mp; a.V = sh.V; a.v0 = 0; a.steps = sh.panels;
        a.part = f.part; a.tlogit = f.tlogit; a.v_shares = ce_logit_shares(sh, sh.Vp);
        if ((rc = ce_logits<T, SPLIT, false>(a, sh.Vp, ce_big(sh), (const T *)p->bias, s))) return rc;
    }
    CeRows r = {};
    r.part = f.part; r.ldp = ce_scores(p) ? (int64_t)CE_SCORE_ROWS : sh.Mp; r.parts = f.parts; r.tlogit = f.tlogit; r.target = p->target;
    r.tc = f.saved.tc; r.orig = f.saved.orig; r.M = p->M; r.V = p->V; r.rsh = ce_rows_shift(p->M, f.parts); r.reduction = p->reduction;
    r.stat = p->saved ? f.saved.stat : nullptr; r.loss = loss; r.sums = f.sums; r.sc = f.saved.sc;
    const int64_t cover = ce_scores(p) ? p->M : sh.Mp;
    const dim3 grid((unsigned)((cover + (1 << r.rsh) - 1) >> r.rsh));
    if (ce_scores(p)) hipLaunchKernelGGL((ce_rows_kernel<false>), grid, dim3(256), 0, s, r);
    else hipLaunchKernelGGL((ce_rows_kernel<true>), grid, dim3(256), 0, s, r);
    TNP_HIP(hipGetLastError());
    return 0;
}

template <typename T, bool SPLIT>
static int ce_backward(const tnp_vocab_ce *p, const CeBackward &b, const float *grad, void *dhidden, void *dweight, void *dbias, hipStream_t s) {
    const CeShape sh = ce_shape(p);
    const CeSaved sv = ce_saved(sh, p->saved);
    int rc;
    if (p->reduction == 0) {
        hipLaunchKernelGGL(ce_gmax_kernel, dim3(1), dim3(1024), 0, s, grad, p->target, p->M, b.up);
        TNP_HIP(hipGetLastError());
    }
    const GemmOperand w{sv.w, sh.Vp, 0}, x{sv.x, sh.Mp, 0};
    for (int k = 0; k < b.pieces; ++k) {
        const int v0 = k * b.piece, cols = sh.Vp - v0 < b.piece ? sh.Vp - v0 : b.piece, live = sh.V - v0 < cols ? sh.V - v0 : cols;
        CeLogits a = {};
        a.w = w; a.x = x; a.sc = sv.sc; a.tc = sv.tc; a.orig = sv.orig; a.xe = sv.xe; a.we = sv.we; a.Mp = sh.Mp; a.V = sh.V; a.v0 = v0; a.steps = sh.panels;
        a.stat = sv.stat; a.grad = p->reduction == 0 ? grad : nullptr; a.up = b.up; a.gs = b.gs; a.xs = b.xs; a.g = b.g; a.g_plane = (int64_t)b.piece * sh.Mp; a.v_shares = ce_logit_shares(sh, cols);
        if ((rc = ce_logits<T, SPLIT, true>(a, cols, ce_big(sh), (const T *)p->bias, s))) return rc;
        const bool last = k == b.pieces - 1;
        const int ks = SPLIT ? 16 : 32;
        CeGrads c = {};
        c.g_plane = (int64_t)b.piece * sh.Mp;
        c.sc = sv.sc; c.grad = grad; c.up = b.up; c.gs = b.gs; c.target = p->target; c.orig = sv.orig; c.M = sh.M; c.reduction = p->reduction; c.D = sh.D;
        c.zero_blocks = dhidden && k == 0 ? (int)(sh.Mp / 64 < 512 ? sh.Mp / 64 : 512) : 0;
        c.x.g = c.w.g = GemmOperand{b.g, sh.Mp, 0};
        c.x.g_panels = c.w.g_panels = cols / ks; c.x.o_panels = c.w.o_panels = sh.panels;
        c.x.o = w; c.x.o.perm = 1; c.x.ok0 = v0; c.x.o_scales = sv.ws + v0;
        c.x.out = dhidden; c.x.part = b.part_x; c.x.part_rows = sh.Mp; c.x.splits = b.splits_x;
        c.x.steps = cols / ks; c.x.add = k > 0;
        c.w.o = x; c.w.o_scales = b.xs ? b.xs : sv.xs;
        c.w.rows = live; c.w.out0 = v0; c.w.out = dweight; c.w.part = b.part_w; c.w.part_rows = b.piece; c.w.splits = b.splits_w;
        c.part_b = dbias ? b.part_b : nullptr; c.ldb = b.piece;
        rc = b.tile == 256 ? ce_launch_grads<T, SPLIT, 256, 256, 2, 4, 4>(c, s) : ce_launch_grads<T, SPLIT, 128, 128, 2, 2, 4>(c, s);
        if (rc) return rc;
        const int ve = sh.D % 4 == 0 ? 4 : 1;
        auto join_blocks = [&](int64_t n) { return (int)std::min<int64_t>((n + 256 * ve - 1) / (256 * ve), CE_JOIN_BLOCKS); };
        const int bx = dhidden && b.part_x && last ? join_blocks(sh.M * sh.D) : 0;
        const int bw = dweight && b.part_w ? join_blocks(c.w.rows * sh.D) : 0, bb = dbias ? (live + 255) / 256 : 0;
        if (bx + bw + bb) {
            T *db = dbias ? (T *)dbias + v0 : nullptr;
            if (ve == 4) hipLaunchKernelGGL((ce_join_kernel<T, 4>), dim3(bx + bw + bb), dim3(256), 0, s, c, bx, bw, live, db);
            else hipLaunchKernelGGL((ce_join_kernel<T, 1>), dim3(bx + bw + bb), dim3(256), 0, s, c, bx, bw, live, db);
            TNP_HIP(hipGetLastError());
        }
    }
    return 0;
}

}  // namespace tnp

using namespace tnp;

extern "C" TNP_API size_t tnp_vocab_ce_saved_bytes(const tnp_vocab_ce *args) {
    if (ce_check(args, "tnp_vocab_ce_saved_bytes")) return 0;
    return ce_saved(ce_shape(args), nullptr).bytes;
}

extern "C" TNP_API size_t tnp_vocab_ce_workspace_bytes(const tnp_vocab_ce *args, int backward) {
    if (ce_check(args, "tnp_vocab_ce_workspace_bytes")) return 0;
    return backward ? ce_backward_layout(args, nullptr).bytes : ce_forward_layout(args, nullptr).bytes;
}

extern "C" TNP_API int tnp_vocab_ce_plan(const tnp_vocab_ce *args, int which) {
    if (ce_check(args, "tnp_vocab_ce_plan")) return -1;
    if (which == TNP_VOCAB_LOGIT_TILE) return ce_scores(args) ? 0 : ce_big(ce_shape(args)) ? 256 : 128;
    if (which == TNP_VOCAB_GRAD_TILE) return ce_backward_layout(args, nullptr).tile;
    if (which == TNP_VOCAB_PIECES) return ce_backward_layout(args, nullptr).pieces;
    TNP_FAIL(-1, "tnp_vocab_ce_plan: unknown question %d", which);
}

extern "C" TNP_API int tnp_vocab_ce_forward(const tnp_vocab_ce *args, float *loss, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = ce_check(args, "tnp_vocab_ce_forward")) return rc;
    if (args->M == 0) TNP_FAIL(-1, "tnp_vocab_ce_forward: no rows");
    if (!args->hidden || !args->weight || !args->target || !loss || !workspace) TNP_FAIL(-1, "tnp_vocab_ce_forward: NULL pointer");
    const CeForward f = ce_forward_layout(args, workspace);
    if (workspace_bytes < f.bytes) TNP_FAIL(-1, "tnp_vocab_ce_forward: workspace of %zu bytes, %zu needed", workspace_bytes, f.bytes);
    hipStream_t s = (hipStream_t)stream;
    if (args->dtype == TNP_F32) return ce_forward<float, 4, true>(args, f, loss, s);
    if (args->dtype == TNP_BF16) return ce_forward<bf16_t, 8, false>(args, f, loss, s);
    return ce_forward<half_t, 8, false>(args, f, loss, s);
}

extern "C" TNP_API int tnp_vocab_ce_backward(const tnp_vocab_ce *args, const float *grad, void *dhidden, void *dweight, void *dbias,
                                             void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = ce_check(args, "tnp_vocab_ce_backward")) return rc;
    if (args->M == 0) TNP_FAIL(-1, "tnp_vocab_ce_backward: no rows");
    if (!args->target || !args->saved || !grad || !workspace) TNP_FAIL(-1, "tnp_vocab_ce_backward: NULL pointer");
    if (dbias && !args->bias) TNP_FAIL(-1, "tnp_vocab_ce_backward: dbias without a bias");
    const CeBackward b = ce_backward_layout(args, workspace);
    if (workspace_bytes < b.bytes) TNP_FAIL(-1, "tnp_vocab_ce_backward: workspace of %zu bytes, %zu needed", workspace_bytes, b.bytes);
    hipStream_t s = (hipStream_t)stream;
    if (args->dtype == TNP_F32) return ce_backward<float, true>(args, b, grad, dhidden, dweight, dbias, s);
    if (args->dtype == TNP_BF16) return ce_backward<bf16_t, false>(args, b, grad, dhidden, dweight, dbias, s);
    return ce_backward<half_t, false>(args, b, grad, dhidden, dweight, dbias, s);
}
