// Token embedding (gfx950): out[i] = scale * weight[token[i]], and the gradient of the table,
//     dweight[v] = scale * sum over { i : token[i] == v } of grad[i]
// summed in an order that the sizes and tokens fix, so that two calls on the same inputs give the same bits.  A negative token is an
// absent track: a zero row forward, nothing backward.  A token >= V has no row: NaN forward (an error that shows and cannot
// fault), nothing backward.
//
// Forward: one pass, bound by memory.  Backward of few tokens: every token's workgroup looks for its like (embed_small_kernel).  Of more:
// the tokens are sorted (a stable radix sort of (token, i) pairs, digits of up to 10 bits), so that all rows of one token are
// neighbours; chunks of 8, 16 or 32 sorted positions are summed by one group of lanes each, whatever the distribution of the tokens.  What
// goes by it is the join of a run over many chunks, one workgroup per run and block of columns: 262144 x 256 bf16 takes 78 us with the tokens
// spread over 65536 rows, 89 with ~ u^6 (the longest run has 41000 rows), 151 with all of them alike.
// Every gradient row is read once and every table row written once; table rows without a token are zeroed by their own workgroups,
// which find them by binary search in the sorted tokens.
#include "vocab_types.h"

namespace tnp {

static constexpr int EMB_SORT_THREADS = 512, EMB_SORT_ROWS = 4;      // eight waves per workgroup of the sort, each with four rows of 64 pairs
static constexpr int EMB_COUNT_ALL = 6;       // workgroups of the sort up to which each counts all keys: 5000 x 64 18.5 us against 20.5, 12000 x 64 22 against 22
                                              // (and a launch less), 16000 x 64 24 against 22
// workgroups of the sort from which on their histograms are summed by segments: 524288 x 64 56 us against 64, 1310720 x 64 163 against 226,
// 16777216 x 16 1.17 ms against 10.7; 128 workgroups (262144 x 64) 48 against 48
static constexpr int EMB_SEGMENTS_FROM = 256;
// Tokens, and elements of the gradient, up to which nothing is sorted.  Tables of 300 rows, all tokens alike / spread, against the sort:
// 36 x 64 9 / 9 us against 16 / 16, 4096 x 64 34 / 10 against 26 / 18, 1024 x 512 17 / 15 against 23 / 17; beyond it: 8192 x 64 spread 24
// against 19, 1024 x 1024 24 / 25 against 22 / 17, 4096 x 512 71 / 55 against 33 / 21.
static constexpr int64_t EMB_SMALL_TOKENS = 4096, EMB_SMALL_ELEMENTS = 1 << 19;
static constexpr int EMB_JOIN_CHUNKS = 32;    // chunks per workgroup of the join
static constexpr int EMB_JOIN_SHORT = 32;     // parts of a run that one group of lanes adds up by itself
static constexpr int EMB_MAX_BITS = 10;      // eight waves' counters of 2^10 digits: 32 KB of LDS
static constexpr int64_t EMB_MAX_TOKENS = 1 << 28;

// ---- forward ----------------------------------------------------------------------------------------------------------------
// 2^lsh lanes per row; U rows per lane whose loads are in flight together (a token without a row loads row 0 and drops it: loads
// under a condition would wait for each other).  43008 x 512 bf16 13.5 us, 4.5 TB/s of tokens, table rows and output (a copy of a GB:
// 5.1); 262144 x 256 bf16 41 us.
template <typename T, int VE, typename I, int U>
__global__ void __launch_bounds__(256) embed_forward_kernel(const I *tokens, int64_t N, const T *weight, int64_t ldw, int64_t V,
                                                            int D, int lsh, float scale, T *out, int64_t ldo) {
    const int lanes = 1 << lsh, rows = 256 >> lsh;
    const int64_t i0 = (int64_t)blockIdx.x * rows * U + (threadIdx.x >> lsh);
    int64_t tok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) tok[u] = i0 + u * rows < N ? (int64_t)tokens[i0 + u * rows] : -1;
    for (int c = (threadIdx.x & (lanes - 1)) * VE; c < D; c += lanes * VE) {
        Pack<T, VE> w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = *(const Pack<T, VE> *)(weight + (tok[u] >= 0 && tok[u] < V ? tok[u] : 0) * ldw + c);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * rows >= N) continue;
#pragma unroll
            for (int e = 0; e < VE; ++e)
                w[u].v[e] = from_f32<T>(tok[u] < 0 ? 0.0f : tok[u] < V ? to_f32(w[u].v[e]) * scale : __builtin_nanf(""));
            *(Pack<T, VE> *)(out + (i0 + u * rows) * ldo + c) = w[u];
        }
    }
}

// ---- stable radix sort of (token, i) ----------------------------------------------------------------------------------------
// Keys: the token, or V for a token outside the table (sorted behind everything, skipped by the sums).  Bound by latency, not bytes: a
// pass over 43008 tokens takes 5.3 us of counting and 9.6 of scattering, over 262144 (17-bit keys, two passes) 4.8 and 16.
template <typename I>
__device__ __forceinline__ uint32_t embed_key(const I *tokens, const uint32_t *keys, int64_t i, uint32_t V) {
    if (keys) return keys[i];
    const int64_t t = (int64_t)tokens[i];
    return t < 0 || t >= (int64_t)V ? V : (uint32_t)t;
}

// lanes of the wave that hold the same digit, among the lanes with `live`
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits, bool live) {
    uint64_t m = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const bool one = (d >> b) & 1;
        const uint64_t v = __ballot(one);
        m &= one ? v : ~v;
    }
    return m;
}

// Ranks of a wave's pairs within (wave, digit), in ascending position, counts left in cnt[] (this wave's counters, zeroed by the
// caller).  Only the first lane of a digit's group touches the counter, and LDS operations of a wave execute in order.
template <typename I, bool RANK>
__device__ __forceinline__ void embed_count(const I *tokens, const uint32_t *keys, int64_t base, int64_t N, uint32_t V, int shift,
                                            int bits, uint32_t *cnt, uint32_t *key, uint32_t *rank) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < EMB_SORT_ROWS; ++r) {
        const int64_t i = base + r * 64 + lane;
        key[r] = i < N ? embed_key(tokens, keys, i, V) : 0;
    }
#pragma unroll
    for (int r = 0; r < EMB_SORT_ROWS; ++r) {
        const bool live = base + r * 64 + lane < N;
        const uint32_t d = (key[r] >> shift) & ((1u << bits) - 1);
        const uint64_t m = same_digit(d, bits, live);
        const int first = __ffsll((unsigned long long)m) - 1;
        uint32_t before = 0;
        if (live && lane == first) before = atomicAdd(&cnt[d], (uint32_t)__popcll(m));
        if (RANK) rank[r] = __shfl(before, first & 63) + (uint32_t)__popcll(m & ((1ull << lane) - 1));
    }
}

template <typename I>
__global__ void __launch_bounds__(EMB_SORT_THREADS) embed_hist_kernel(const I *tokens, const uint32_t *keys, int64_t N, uint32_t V,
                                                                      int shift, int bits, uint32_t *hist) {
    extern __shared__ uint32_t cnt[];
    const int nb = 1 << bits;
    for (int b = threadIdx.x; b < nb; b += EMB_SORT_THREADS) cnt[b] = 0;
    __syncthreads();
    uint32_t key[EMB_SORT_ROWS];
    const int64_t base = ((int64_t)blockIdx.x * (EMB_SORT_THREADS / 64) + (threadIdx.x >> 6)) * (EMB_SORT_ROWS * 64);
    embed_count<I, false>(tokens, keys, base, N, V, shift, bits, cnt, key, nullptr);
    __syncthreads();
    for (int b = threadIdx.x; b < nb; b += EMB_SORT_THREADS) hist[(size_t)blockIdx.x * nb + b] = cnt[b];
}

// sums of 2^sl histograms each
__global__ void __launch_bounds__(256) embed_segments_kernel(const uint32_t *hist, int nblk, int nb, int sl, uint32_t *seg) {
    const int b = blockIdx.y * 256 + threadIdx.x, k0 = blockIdx.x << sl, k1 = min(k0 + (1 << sl), nblk);
    if (b >= nb) return;
    constexpr int U = 16;
    uint32_t sum = 0;
    for (int k = k0; k < k1; k += U) {
        uint32_t h[U];
#pragma unroll
        for (int u = 0; u < U; ++u) h[u] = hist[(size_t)(k + u < k1 ? k + u : k) * nb + b];
#pragma unroll
        for (int u = 0; u < U; ++u) sum += k + u < k1 ? h[u] : 0;
    }
    seg[(size_t)blockIdx.x * nb + b] = sum;
}

// Every workgroup forms its own offsets from the histograms of all of them (nblk * 2^bits counters, L2-resident): one launch less
// per pass than a scan kernel in between.  Up to six workgroups (hist == NULL) count all the keys themselves, another launch less.
// From 256 on the histograms are summed by segments first (seg): what all workgroups read together would grow with their square.
template <typename I>
__global__ void __launch_bounds__(EMB_SORT_THREADS) embed_scatter_kernel(const I *tokens, const uint32_t *keys, const uint32_t *idx,
                                                                         int64_t N, uint32_t V, int shift, int bits,
                                                                         const uint32_t *hist, const uint32_t *seg, int sl, int nblk,
                                                                         uint32_t *keys_out, uint32_t *idx_out) {
    extern __shared__ uint32_t lds[];
    const int nb = 1 << bits, nw = EMB_SORT_THREADS / 64;
    uint32_t *cnt = lds;                // [waves][nb]: counts, then the first position of (wave, digit)
    uint32_t *part = lds + nw * nb;     // [waves] sums of the scan over digits
    uint32_t *all = part + nw;          // [2][nb] without histograms: keys of the digit, those of them before this workgroup's
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    for (int b = tid; b < nw * nb; b += EMB_SORT_THREADS) cnt[b] = 0;
    const bool count_all = nblk > 1 && !hist;
    if (count_all)
        for (int b = tid; b < 2 * nb; b += EMB_SORT_THREADS) all[b] = 0;
    __syncthreads();
    if (count_all) {
        const int64_t mine = (int64_t)blockIdx.x * nw * EMB_SORT_ROWS * 64;
        constexpr int U = 8;
        for (int64_t i = tid; i < N; i += EMB_SORT_THREADS * U) {
            uint32_t k[U];
#pragma unroll
            for (int u = 0; u < U; ++u) k[u] = i + u * EMB_SORT_THREADS < N ? embed_key(tokens, keys, i + u * EMB_SORT_THREADS, V) : 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u * EMB_SORT_THREADS >= N) continue;
                const uint32_t d = (k[u] >> shift) & (nb - 1);
                atomicAdd(&all[d], 1u);
                if (i + u * EMB_SORT_THREADS < mine) atomicAdd(&all[nb + d], 1u);
            }
        }
    }
    uint32_t key[EMB_SORT_ROWS], rank[EMB_SORT_ROWS], from[EMB_SORT_ROWS];
    const int64_t base = ((int64_t)blockIdx.x * nw + wave) * (EMB_SORT_ROWS * 64);
#pragma unroll
    for (int r = 0; r < EMB_SORT_ROWS; ++r) {
        const int64_t i = base + r * 64 + lane;
        from[r] = idx && i < N ? idx[i] : (uint32_t)i;
    }
    embed_count<I, true>(tokens, keys, base, N, V, shift, bits, cnt + wave * nb, key, rank);
    __syncthreads();
    const int per = (nb + EMB_SORT_THREADS - 1) / EMB_SORT_THREADS;       // digits per thread: 1 or 2
    uint32_t total[2] = {0, 0}, before[2] = {0, 0}, sum = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int b = tid * per + j;
        if (j >= per || b >= nb) continue;
        if (nblk == 1) {
            for (int w = 0; w < nw; ++w) total[j] += cnt[w * nb + b];
        } else if (count_all) {
            total[j] = all[b];
            before[j] = all[nb + b];
        } else {
            constexpr int U = 16;                              // counters in flight
            auto add = [&](const uint32_t *from, int k0, int k1, int mine) {      // total += all of them, before += those below mine
                for (int k = k0; k < k1; k += U) {
                    uint32_t h[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) h[u] = k + u < k1 ? from[(size_t)(k + u) * nb + b] : 0;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        before[j] += k + u < mine ? h[u] : 0;
                        total[j] += h[u];
                    }
                }
            };
            if (!seg) {
                add(hist, 0, nblk, blockIdx.x);
            } else {
                const int s = blockIdx.x >> sl;
                add(hist, s << sl, blockIdx.x, blockIdx.x);
                total[j] = 0;
                add(seg, 0, (nblk + (1 << sl) - 1) >> sl, s);
            }
        }
        sum += total[j];
    }
    uint32_t incl = sum;                                       // inclusive scan over the wave, then over the waves
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t v = __shfl_up(incl, off);
        if (lane >= off) incl += v;
    }
    if (lane == 63) part[wave] = incl;
    __syncthreads();
    uint32_t start = incl - sum;
    for (int w = 0; w < wave; ++w) start += part[w];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int b = tid * per + j;
        if (j >= per || b >= nb) continue;
        uint32_t at = start + before[j];
        for (int w = 0; w < nw; ++w) {
            const uint32_t c = cnt[w * nb + b];
            cnt[w * nb + b] = at;
            at += c;
        }
        start += total[j];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < EMB_SORT_ROWS; ++r) {
        const int64_t i = base + r * 64 + lane;
        if (i >= N) continue;
        const uint32_t d = (key[r] >> shift) & (nb - 1);
        const uint32_t at = cnt[wave * nb + d] + rank[r];
        keys_out[at] = key[r];
        idx_out[at] = from[r];
    }
}

// ---- sums over the sorted pairs ---------------------------------------------------------------------------------------------
// first position whose key is > k
__device__ __forceinline__ uint32_t embed_upper(const uint32_t *keys, uint32_t lo, uint32_t hi, uint32_t k) {
    while (lo < hi) {
        const uint32_t mid = lo + ((hi - lo) >> 1);
        if (keys[mid] > k) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// Chunk c = sorted positions [c << csh, (c + 1) << csh), 2^lsh lanes, fp32 sums.  A run (one token) inside the chunk is finished here; the
// part of a run that came in from the chunk before goes to head[c], the first part of a run that goes on into the next to tail[c]
// (embed_join_kernel adds those).  Workgroups from `sum_blocks` on zero the table rows that no token names.  262144 x 256 bf16 into 65536
// rows 46 us, 3.6 TB/s: the gradient's rows are read in the tokens' order, 512 bytes at a time.
template <typename T, int VE>
__global__ void __launch_bounds__(256) embed_reduce_kernel(const uint32_t *keys, const uint32_t *idx, uint32_t N, uint32_t V,
                                                           const T *grad, int64_t ldg, int D, int lsh, int csh, float scale, T *dw,
                                                           int64_t ldd, float *head, float *tail, uint32_t sum_blocks) {
    const int lanes = 1 << lsh;
    if (blockIdx.x >= sum_blocks) {                    // 64 table rows per wave
        const uint32_t v0 = ((blockIdx.x - sum_blocks) * 4 + (threadIdx.x >> 6)) * 64, v = v0 + (threadIdx.x & 63);
        bool none = v < V;
        if (none) {
            const uint32_t at = v == 0 ? 0 : embed_upper(keys, 0, N, v - 1);
            none = at >= N || keys[at] != v;
        }
        uint64_t m = __ballot(none);
        const int c0 = blockIdx.y * lanes * VE;
        const int rows = 64 >> lsh;                    // rows per trip (lsh <= 6)
        const int sub = (threadIdx.x & 63) >> lsh;
        const int c = c0 + (threadIdx.x & (lanes - 1)) * VE;
        while (m) {
            int mine = -1;
            for (int r = 0; r < rows; ++r) {
                const int b = m ? __ffsll((unsigned long long)m) - 1 : -1;
                if (r == sub) mine = b;
                if (m) m &= m - 1;
            }
            if (mine >= 0 && c < D) {
                Pack<T, VE> z;
#pragma unroll
                for (int e = 0; e < VE; ++e) z.v[e] = from_f32<T>(0.0f);
                *(Pack<T, VE> *)(dw + (int64_t)(v0 + mine) * ldd + c) = z;
            }
        }
        return;
    }
    const uint32_t chunk = blockIdx.x * (256u >> lsh) + (threadIdx.x >> lsh);
    const uint64_t a64 = (uint64_t)chunk << csh;
    if (a64 >= N) return;
    const uint32_t a = (uint32_t)a64, b = min(a + (1u << csh), N);
    const int c = (blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * VE;
    if (c >= D) return;
    uint32_t cur = keys[a];
    bool incoming = a > 0 && keys[a - 1] == cur;
    float acc[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
    auto part = [&](float *where) {
#pragma unroll
        for (int e = 0; e < VE; ++e) where[(size_t)chunk * D + c + e] = acc[e];
    };
    auto finish = [&]() {
        Pack<T, VE> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) o.v[e] = from_f32<T>(acc[e] * scale);
        *(Pack<T, VE> *)(dw + (int64_t)cur * ldd + c) = o;
    };
    constexpr int U = 8;                               // rows in flight
    for (uint32_t p = a; p < b; p += U) {
        uint32_t k[U];
        Pack<T, VE> g[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {                  // behind the chunk: its last row again, not added
            const uint32_t at = p + u < b ? p + u : b - 1;
            k[u] = keys[at];
            g[u] = *(const Pack<T, VE> *)(grad + (int64_t)idx[at] * ldg + c);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p + u >= b) break;
            if (k[u] != cur) {
                if (incoming) part(head); else finish();
                incoming = false;
                cur = k[u];
#pragma unroll
                for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
            }
            if (cur >= V) return;                      // only tokens outside the table are left
#pragma unroll
            for (int e = 0; e < VE; ++e) acc[e] += to_f32(g[u].v[e]);
        }
    }
    if (cur >= V) return;
    const bool goes_on = b < N && keys[b] == cur;
    if (incoming) part(head);
    else if (goes_on) part(tail);
    else finish();
}

// VE partial sums (rows of D floats, D a multiple of VE)
template <int VE> struct Parts { Pack<float, (VE < 4 ? VE : 4)> p[VE < 4 ? 1 : VE / 4]; };
template <int VE> __device__ __forceinline__ Parts<VE> load_parts(const float *at) {
    Parts<VE> r;
#pragma unroll
    for (int k = 0; k < (VE < 4 ? 1 : VE / 4); ++k) r.p[k] = *(const Pack<float, (VE < 4 ? VE : 4)> *)(at + 4 * k);
    return r;
}

// Runs that go on past their chunk: tail[c] + head[c + 1] + ... of the run that starts in chunk c.  A workgroup looks after 32 chunks:
// first every group of lanes adds up runs of up to 32 parts by itself, then all of them together stride over each longer one and
// meet in LDS.  Every order of addition is fixed by the sizes.  262144 x 256 bf16, tokens ~ u^6: 23 us (the longest run has 41000 rows);
// 43008 x 64 into 257 rows 9.6 us.
template <typename T, int VE>
__global__ void __launch_bounds__(512) embed_join_kernel(const uint32_t *keys, uint32_t N, uint32_t V, int D, int lsh, int csh, float scale,
                                                         T *dw, int64_t ldd, const float *head, const float *tail) {
    extern __shared__ float sums[];                    // [512][VE]
    __shared__ uint32_t long_chunk[EMB_JOIN_CHUNKS];
    __shared__ int longs;
    const int lanes = 1 << lsh, groups = 512 >> lsh, grp = threadIdx.x >> lsh;
    const int c = (blockIdx.y * lanes + (threadIdx.x & (lanes - 1))) * VE;
    if (threadIdx.x < 64) {                            // the first wave looks for the runs
        const uint64_t chunk = (uint64_t)blockIdx.x * EMB_JOIN_CHUNKS + threadIdx.x, a = chunk << csh, b = (chunk + 1) << csh;
        bool starts = false, more = false;
        if (threadIdx.x < EMB_JOIN_CHUNKS && b < N) {
            const uint32_t k = keys[b - 1];
            starts = k < V && keys[b] == k && !(a > 0 && keys[a - 1] == k);
            const uint64_t far = b + ((uint64_t)EMB_JOIN_SHORT << csh);
            more = starts && far < N && keys[far] == k;
        }
        const uint64_t m = __ballot(more), s = __ballot(starts);
        if (threadIdx.x < EMB_JOIN_CHUNKS) {
            long_chunk[threadIdx.x] = starts ? (more ? 2u : 1u) : 0u;
            if (threadIdx.x == 0) longs = s ? __popcll(m) : -1;
        }
    }
    __syncthreads();
    if (longs < 0) return;
    auto finish = [&](uint32_t k, const float *acc) {
        Pack<T, VE> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) o.v[e] = from_f32<T>(acc[e] * scale);
        *(Pack<T, VE> *)(dw + (int64_t)k * ldd + c) = o;
    };
    for (int j = grp; j < EMB_JOIN_CHUNKS; j += groups) {
        if (long_chunk[j] != 1 || c >= D) continue;
        const uint32_t chunk = blockIdx.x * EMB_JOIN_CHUNKS + j, b = (chunk + 1) << csh, k = keys[b];
        // parts behind the run's end: the run's first part again, not added -- loads under a condition wait for each other
        const Parts<VE> t = load_parts<VE>(tail + (size_t)chunk * D + c);
        float acc[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] = t.p[e / 4].v[e % 4];
        constexpr int P = 16, U = 8;                   // keys looked at and parts fetched at a time
        for (int q0 = 0, parts = P; q0 < EMB_JOIN_SHORT && parts == P; q0 += P) {
            const uint64_t b0 = (uint64_t)b + ((uint64_t)q0 << csh);
            uint32_t first[P];
#pragma unroll
            for (int u = 0; u < P; ++u) first[u] = keys[b0 + (u << csh) < N ? b0 + (u << csh) : b - 1];
            parts = 0;
#pragma unroll
            for (int u = 0; u < P; ++u) parts += b0 + (u << csh) < N && first[u] == k;
            for (int q = 0; q < parts; q += U) {
                Parts<VE> h[U];
#pragma unroll
                for (int u = 0; u < U; ++u) h[u] = load_parts<VE>(head + (size_t)(chunk + 1 + (q + u < parts ? q0 + q + u : 0)) * D + c);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int e = 0; e < VE; ++e) acc[e] += q + u < parts ? h[u].p[e / 4].v[e % 4] : 0.0f;
            }
        }
        finish(k, acc);
    }
    if (longs == 0) return;
    for (int j = 0; j < EMB_JOIN_CHUNKS; ++j) {
        if (long_chunk[j] != 2) continue;              // the same for the whole workgroup
        const uint32_t chunk = blockIdx.x * EMB_JOIN_CHUNKS + j, k = keys[(chunk + 1) << csh];
        // last chunk that the run enters: it begins with k (monotone in the chunk), 512 probes at a time
        uint32_t last = chunk + 1 + EMB_JOIN_SHORT, end = (N + (1u << csh) - 1) >> csh;
        while (end - last > 1) {
            const uint32_t step = (end - last + 511) / 512;
            const uint64_t at = last + (uint64_t)(threadIdx.x + 1) * step;
            const uint32_t hit = (uint32_t)__syncthreads_count(at < end && keys[at << csh] == k);
            last += hit * step;
            end = min(last + step, end);
        }
        float acc[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] = grp == 0 && c < D ? tail[(size_t)chunk * D + c + e] : 0.0f;
        if (c < D) {
            constexpr int U = 8;
            for (uint32_t q = chunk + 1 + grp; q <= last; q += groups * U) {
                Parts<VE> h[U];
#pragma unroll
                for (int u = 0; u < U; ++u) h[u] = load_parts<VE>(head + (size_t)(q + u * groups <= last ? q + u * groups : q) * D + c);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int e = 0; e < VE; ++e) acc[e] += q + u * groups <= last ? h[u].p[e / 4].v[e % 4] : 0.0f;
            }
        }
        __syncthreads();                               // the sums of the run before have been read
#pragma unroll
        for (int e = 0; e < VE; ++e) sums[threadIdx.x * VE + e] = acc[e];
        __syncthreads();
        if (grp == 0 && c < D) {
            for (int g = 1; g < groups; ++g)
#pragma unroll
                for (int e = 0; e < VE; ++e) acc[e] += sums[(g * lanes + threadIdx.x) * VE + e];
            finish(k, acc);
        }
    }
}

// ---- few tokens: no sort ----------------------------------------------------------------------------------------------------
// One launch: workgroup (i < N, 64 columns) owns token i's row if no earlier position names it, lists the positions that do (every wave
// compacts its quarter of them in order) and adds their gradient rows, groups of lanes striding over the list; the workgroups behind
// zero 256 table rows each, less those named.  N^2 comparisons from the L2 instead of four to six dependent launches.  Bound by the
// token whose list is longest, which is why a workgroup takes 64 columns only.
template <typename T, int VE, typename I>
__global__ void __launch_bounds__(256) embed_small_kernel(const I *tokens, int N, int64_t V, const T *grad, int64_t ldg, int D, float scale,
                                                          T *dw, int64_t ldd) {
    constexpr int LANES = 64 / VE, GROUPS = 256 / LANES, U = 8;
    __shared__ uint16_t list[4][EMB_SMALL_TOKENS / 4];
    __shared__ int count[4];
    __shared__ float sums[256 * VE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, grp = tid / LANES;
    const int c = ((int)blockIdx.y * LANES + tid % LANES) * VE;
    if ((int)blockIdx.x >= N) {
        uint8_t *named = (uint8_t *)list;
        const int64_t v0 = (int64_t)(blockIdx.x - N) * 256;
        named[tid] = 0;
        __syncthreads();
        for (int j = tid; j < N; j += 256 * U) {
            int64_t t[U];
#pragma unroll
            for (int u = 0; u < U; ++u) t[u] = tokens[j + u * 256 < N ? j + u * 256 : j];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (t[u] >= v0 && t[u] < v0 + 256) named[t[u] - v0] = 1;
        }
        __syncthreads();
        if (c >= D) return;
        Pack<T, VE> z;
#pragma unroll
        for (int e = 0; e < VE; ++e) z.v[e] = from_f32<T>(0.0f);
        for (int r = grp; r < 256 && v0 + r < V; r += GROUPS)
            if (!named[r]) *(Pack<T, VE> *)(dw + (v0 + r) * ldd + c) = z;
        return;
    }
    const int i = blockIdx.x;
    const int64_t t = tokens[i];
    if (t < 0 || t >= V) return;                       // uniform
    bool before = false;
    for (int j = tid; j < i; j += 256 * U) {
        int64_t o[U];
#pragma unroll
        for (int u = 0; u < U; ++u) o[u] = tokens[j + u * 256 < i ? j + u * 256 : j];
#pragma unroll
        for (int u = 0; u < U; ++u) before = before || o[u] == t;
    }
    if (__syncthreads_or(before)) return;
    const int quarter = (N - i + 3) / 4, j0 = i + wave * quarter, j1 = j0 + quarter < N ? j0 + quarter : N;
    int n = 0;
    for (int j = j0; j < j1; j += 64 * U) {
        int64_t o[U];
#pragma unroll
        for (int u = 0; u < U; ++u) o[u] = tokens[j + u * 64 + lane < j1 ? j + u * 64 + lane : i];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool hit = j + u * 64 + lane < j1 && o[u] == t;
            const uint64_t m = __ballot(hit);
            if (hit) list[wave][n + __popcll(m & ((1ull << lane) - 1))] = (uint16_t)(j + u * 64 + lane);
            n += __popcll(m);
        }
    }
    if (lane == 0) count[wave] = n;
    __syncthreads();
    const int n1 = count[0], n2 = n1 + count[1], n3 = n2 + count[2], all = n3 + count[3];
    auto at = [&](int k) -> int64_t { return k < n1 ? list[0][k] : k < n2 ? list[1][k - n1] : k < n3 ? list[2][k - n2] : list[3][k - n3]; };
    float acc[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] = 0.0f;
    if (c < D)
        for (int k = grp; k < all; k += GROUPS * U) {
            Pack<T, VE> g[U];
#pragma unroll
            for (int u = 0; u < U; ++u) g[u] = *(const Pack<T, VE> *)(grad + at(k + u * GROUPS < all ? k + u * GROUPS : k) * ldg + c);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < VE; ++e) acc[e] += k + u * GROUPS < all ? to_f32(g[u].v[e]) : 0.0f;
        }
    const int used = all < GROUPS ? all : GROUPS;      // groups that have a row
    if (used > 1) {
#pragma unroll
        for (int e = 0; e < VE; ++e) sums[tid * VE + e] = acc[e];
        __syncthreads();
    }
    if (grp == 0 && c < D) {
        for (int g = 1; g < used; ++g)
#pragma unroll
            for (int e = 0; e < VE; ++e) acc[e] += sums[(g * LANES + tid) * VE + e];
        Pack<T, VE> o;
#pragma unroll
        for (int e = 0; e < VE; ++e) o.v[e] = from_f32<T>(acc[e] * scale);
        *(Pack<T, VE> *)(dw + t * ldd + c) = o;
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------
// elements per lane: 16 bytes where rows and pointers allow it, else 4, else one element
static int embed_width(int dtype, int D, std::initializer_list<int64_t> lds, std::initializer_list<const void *> ptrs) {
    const int sz = (int)dtype_bytes(dtype);
    for (int bytes : {16, 4}) {
        const int ve = bytes / sz;
        bool ok = D % ve == 0;
        for (int64_t ld : lds) ok = ok && ld % ve == 0;
        for (const void *p : ptrs) ok = ok && (uintptr_t)p % bytes == 0;
        if (ok) return ve;
    }
    return 1;
}

static int lane_shift(int D, int ve, int most) {
    int s = 0;
    while (s < most && ((int64_t)ve << s) < D) ++s;
    return s;
}

struct EmbedSort { int bits, passes, nblk, sl, nseg; };  // nseg sums of 2^sl histograms, or 0
static EmbedSort embed_sort_plan(int64_t N, int64_t V) {
    EmbedSort p = {};
    int need = 1;
    while (((int64_t)1 << need) <= V) ++need;          // keys 0 .. V
    p.passes = (need + EMB_MAX_BITS - 1) / EMB_MAX_BITS;
    p.bits = (need + p.passes - 1) / p.passes;
    const int64_t items = EMB_SORT_THREADS * EMB_SORT_ROWS;
    p.nblk = (int)((N + items - 1) / items);
    p.sl = 6;                                          // about as many sums as histograms in one
    while (((int64_t)1 << 2 * p.sl) < p.nblk) ++p.sl;
    p.nseg = p.nblk >= EMB_SEGMENTS_FROM ? (p.nblk + (1 << p.sl) - 1) >> p.sl : 0;
    return p;
}

static bool embed_small(int64_t N, int D) { return N <= EMB_SMALL_TOKENS && N * D <= EMB_SMALL_ELEMENTS; }

// rows of head / tail: chunks are shorter than 32 positions only where there are fewer than 1024 * 64 of the shorter ones
static size_t embed_parts(int64_t N) {
    const size_t most = (size_t)((N + 31) / 32), short_ones = (size_t)((N + 7) / 8);
    return most > 131072 ? most : short_ones < 131072 ? short_ones : 131072;
}

static inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename T, int VE, typename I>
static int embed_forward_run(const I *tokens, int64_t N, const T *w, int64_t ldw, int64_t V, int D, float scale, T *out, int64_t ldo,
                             hipStream_t s) {
    const int lsh = lane_shift(D, VE, 8);
    const int64_t rows = 256 >> lsh;
    // four rows per lane once one row per lane would be several rounds of workgroups: 1048576 x 64 fp32 75 us against 86, 16384 x 64 9.8
    // against 8.9
    const bool four = N / rows >= 4096;
    const int64_t most = rows << 22;                   // rows per launch: a grid holds fewer than 2^32 threads
    for (int64_t i = 0; i < N; i += most) {
        const int64_t n = N - i < most ? N - i : most, per = four ? rows * 4 : rows;
        const dim3 grid((unsigned)((n + per - 1) / per));
        if (four)
            hipLaunchKernelGGL((embed_forward_kernel<T, VE, I, 4>), grid, dim3(256), 0, s, tokens + i, n, w, ldw, V, D, lsh, scale,
                               out + i * ldo, ldo);
        else
            hipLaunchKernelGGL((embed_forward_kernel<T, VE, I, 1>), grid, dim3(256), 0, s, tokens + i, n, w, ldw, V, D, lsh, scale,
                               out + i * ldo, ldo);
        TNP_HIP(hipGetLastError());
    }
    return 0;
}

template <typename T, int VE>
static int embed_forward_typed(const void *tokens, int tb, int64_t N, const void *w, int64_t ldw, int64_t V, int D, float scale, void *out,
                               int64_t ldo, hipStream_t s) {
    if (tb == 8) return embed_forward_run<T, VE, int64_t>((const int64_t *)tokens, N, (const T *)w, ldw, V, D, scale, (T *)out, ldo, s);
    return embed_forward_run<T, VE, int32_t>((const int32_t *)tokens, N, (const T *)w, ldw, V, D, scale, (T *)out, ldo, s);
}

template <typename I>
static int embed_sort(const I *tokens, int64_t N, uint32_t V, const EmbedSort &p, uint32_t *keys[2], uint32_t *idx[2], uint32_t *hist,
                      hipStream_t s) {
    for (int pass = 0; pass < p.passes; ++pass) {
        const uint32_t *kin = pass ? keys[(pass + 1) & 1] : nullptr, *iin = pass ? idx[(pass + 1) & 1] : nullptr;
        const size_t nb = (size_t)1 << p.bits;
        const bool count_all = p.nblk <= EMB_COUNT_ALL;
        if (!count_all) {
            hipLaunchKernelGGL((embed_hist_kernel<I>), dim3(p.nblk), dim3(EMB_SORT_THREADS), nb * 4, s, tokens, kin, N, V, pass * p.bits,
                               p.bits, hist);
            TNP_HIP(hipGetLastError());
        }
        uint32_t *seg = p.nseg ? hist + (size_t)p.nblk * nb : nullptr;
        if (seg) {
            hipLaunchKernelGGL(embed_segments_kernel, dim3(p.nseg, (unsigned)((nb + 255) / 256)), dim3(256), 0, s, hist, p.nblk, (int)nb, p.sl,
                               seg);
            TNP_HIP(hipGetLastError());
        }
        const size_t smem = (EMB_SORT_THREADS / 64 * nb + EMB_SORT_THREADS / 64 + (count_all ? 2 * nb : 0)) * 4;
        hipLaunchKernelGGL((embed_scatter_kernel<I>), dim3(p.nblk), dim3(EMB_SORT_THREADS), smem, s, tokens, kin, iin, N, V, pass * p.bits,
                           p.bits, count_all ? nullptr : hist, seg, p.sl, p.nblk, keys[pass & 1], idx[pass & 1]);
        TNP_HIP(hipGetLastError());
    }
    return 0;
}

template <typename T, int VE>
static int embed_sums(const uint32_t *keys, const uint32_t *idx, uint32_t N, uint32_t V, const T *grad, int64_t ldg, int D, float scale, T *dw,
                      int64_t ldd, float *head, float *tail, hipStream_t s) {
    const int lsh = lane_shift(D, VE, 6);
    const unsigned cols = (unsigned)((D + (VE << lsh) - 1) / (VE << lsh));
    // 32 positions per chunk where that already is a wave per SIMD; shorter chunks shorten the chain of dependent loads of a small
    // batch (43008 x 64: 6 us at 8 positions, 16 at 32)
    int csh = 5;
    while (csh > 3 && (((uint64_t)N >> csh << lsh) >> 6) * cols < 1024) --csh;
    const unsigned chunks = (unsigned)(((uint64_t)N + (1u << csh) - 1) >> csh);
    const unsigned sum_blocks = (unsigned)(((uint64_t)chunks + (256u >> lsh) - 1) / (256u >> lsh));
    const unsigned zero_blocks = (unsigned)(((uint64_t)V + 255) / 256);
    hipLaunchKernelGGL((embed_reduce_kernel<T, VE>), dim3(sum_blocks + zero_blocks, cols), dim3(256), 0, s, keys, idx, N, V, grad, ldg, D, lsh,
                       csh, scale, dw, ldd, head, tail, sum_blocks);
    TNP_HIP(hipGetLastError());
    if (chunks > 1) {
        hipLaunchKernelGGL((embed_join_kernel<T, VE>), dim3((chunks + EMB_JOIN_CHUNKS - 1) / EMB_JOIN_CHUNKS, cols), dim3(512), 512 * VE * 4, s,
                           keys, N, V, D, lsh, csh, scale, dw, ldd, head, tail);
        TNP_HIP(hipGetLastError());
    }
    return 0;
}

}  // namespace tnp

using namespace tnp;

static int embed_check(const char *who, int token_bytes, int64_t N, int64_t V, int D, int dtype, int64_t ld1, int64_t ld2) {
    if (token_bytes != 4 && token_bytes != 8) TNP_FAIL(-1, "%s: tokens are int32 or int64 (got %d bytes)", who, token_bytes);
    if (!dtype_known(dtype)) TNP_FAIL(-1, "%s: unknown dtype %d", who, dtype);
    if (N < 0 || N > EMB_MAX_TOKENS) TNP_FAIL(-1, "%s: %lld tokens (0 .. 2^28)", who, (long long)N);
    if (V < 1 || V > (1 << 30) || D < 1 || D > (1 << 20)) TNP_FAIL(-1, "%s: table of %lld x %d", who, (long long)V, D);
    if (ld1 < D || ld2 < D) TNP_FAIL(-1, "%s: a row stride is smaller than the %d columns", who, D);
    return 0;
}

#define TNP_BY_WIDTH(FN, ve, dtype, ...)                                                                                   \
    ((dtype) == TNP_F32 ? ((ve) == 4 ? FN<float, 4>(__VA_ARGS__) : FN<float, 1>(__VA_ARGS__))                               \
     : (dtype) == TNP_BF16 ? ((ve) == 8 ? FN<bf16_t, 8>(__VA_ARGS__) : (ve) == 2 ? FN<bf16_t, 2>(__VA_ARGS__) : FN<bf16_t, 1>(__VA_ARGS__)) \
                           : ((ve) == 8 ? FN<half_t, 8>(__VA_ARGS__) : (ve) == 2 ? FN<half_t, 2>(__VA_ARGS__) : FN<half_t, 1>(__VA_ARGS__)))

extern "C" TNP_API int tnp_token_embedding_forward(const void *tokens, int token_bytes, int64_t N, const void *weight, int64_t ldw, int64_t V,
                                                   int D, int dtype, float scale, void *out, int64_t ldo, void *stream) {
    if (int rc = embed_check("tnp_token_embedding_forward", token_bytes, N, V, D, dtype, ldw, ldo)) return rc;
    if (N == 0) return 0;
    if (!tokens || !weight || !out) TNP_FAIL(-1, "tnp_token_embedding_forward: NULL pointer");
    const int ve = embed_width(dtype, D, {ldw, ldo}, {weight, out});
    return TNP_BY_WIDTH(embed_forward_typed, ve, dtype, tokens, token_bytes, N, weight, ldw, V, D, scale, out, ldo, (hipStream_t)stream);
}

extern "C" TNP_API size_t tnp_token_embedding_backward_workspace_bytes(int64_t N, int64_t V, int D) {
    if (V < 1 || D < 1 || embed_small(N, D)) return 0;
    const EmbedSort p = embed_sort_plan(N, V);
    const size_t chunks = embed_parts(N);
    return 4 * up256((size_t)N * 4) + up256((size_t)(p.nblk + p.nseg) * 4 << p.bits) + 2 * up256(chunks * (size_t)D * 4);
}

namespace tnp {
template <typename T, int VE>
static int embed_backward_typed(const uint32_t *keys, const uint32_t *idx, int64_t N, int64_t V, const void *grad, int64_t ldg, int D, float scale,
                                void *dw, int64_t ldd, float *head, float *tail, hipStream_t s) {
    return embed_sums<T, VE>(keys, idx, (uint32_t)N, (uint32_t)V, (const T *)grad, ldg, D, scale, (T *)dw, ldd, head, tail, s);
}
template <typename T, int VE>
static int embed_small_typed(const void *tokens, int tb, int64_t N, int64_t V, const void *grad, int64_t ldg, int D, float scale, void *dw,
                             int64_t ldd, hipStream_t s) {
    const dim3 grid((unsigned)(N + (V + 255) / 256), (unsigned)((D + 63) / 64));
    if (tb == 8) hipLaunchKernelGGL((embed_small_kernel<T, VE, int64_t>), grid, dim3(256), 0, s, (const int64_t *)tokens, (int)N, V,
                                    (const T *)grad, ldg, D, scale, (T *)dw, ldd);
    else hipLaunchKernelGGL((embed_small_kernel<T, VE, int32_t>), grid, dim3(256), 0, s, (const int32_t *)tokens, (int)N, V, (const T *)grad, ldg,
                            D, scale, (T *)dw, ldd);
    TNP_HIP(hipGetLastError());
    return 0;
}
}  // namespace tnp

extern "C" TNP_API int tnp_token_embedding_backward(const void *tokens, int token_bytes, int64_t N, const void *grad, int64_t ldg, int64_t V,
                                                    int D, int dtype, float scale, void *dweight, int64_t ldd, void *workspace,
                                                    size_t workspace_bytes, void *stream) {
    if (int rc = embed_check("tnp_token_embedding_backward", token_bytes, N, V, D, dtype, ldg, ldd)) return rc;
    if (!dweight || (N > 0 && (!tokens || !grad))) TNP_FAIL(-1, "tnp_token_embedding_backward: NULL pointer");
    hipStream_t s = (hipStream_t)stream;
    const int ve = embed_width(dtype, D, {ldg, ldd}, {grad, dweight});
    if (embed_small(N, D))
        return TNP_BY_WIDTH(embed_small_typed, ve, dtype, tokens, token_bytes, N, V, grad, ldg, D, scale, dweight, ldd, s);
    const size_t need = tnp_token_embedding_backward_workspace_bytes(N, V, D);
    if (!workspace || workspace_bytes < need) TNP_FAIL(-1, "tnp_token_embedding_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    uint32_t *keys[2], *idx[2];
    const EmbedSort p = embed_sort_plan(N, V);
    char *w = (char *)workspace;
    for (int k = 0; k < 2; ++k) { keys[k] = (uint32_t *)w; w += up256((size_t)N * 4); idx[k] = (uint32_t *)w; w += up256((size_t)N * 4); }
    uint32_t *hist = (uint32_t *)w;
    w += up256((size_t)(p.nblk + p.nseg) * 4 << p.bits);
    float *head = (float *)w, *tail = (float *)(w + up256(embed_parts(N) * D * 4));
    const int rc = token_bytes == 8 ? embed_sort((const int64_t *)tokens, N, (uint32_t)V, p, keys, idx, hist, s)
                                    : embed_sort((const int32_t *)tokens, N, (uint32_t)V, p, keys, idx, hist, s);
    if (rc) return rc;
    const int at = (p.passes - 1) & 1;
    return TNP_BY_WIDTH(embed_backward_typed, ve, dtype, keys[at], idx[at], N, V, grad, ldg, D, scale, dweight, ldd, head, tail, s);
}
