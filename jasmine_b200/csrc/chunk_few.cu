// Attention of a few new tokens of each sequence over a paged cache (bf16 or 8-bit): single tokens, drafts being verified.  Up to 16 rows of queries
// (tokens x query heads of a kv head) share every cached byte, so the kernel is bound by the bytes of the cache; more rows are groups of tokens that read the cache once each.
//
// All pages that any (sequence, kv head, group) sees are one row of work, cut into equal runs, one per CTA: as many CTAs as the chip holds, each with the same number of bytes
// however ragged the contexts are.  A run holds the end of one (sequence, kv head, group), perhaps whole ones, and the beginning of another: at most two partial results per
// CTA, so the scratch does not grow with contexts or sequences.  A producer thread keeps a ring of pages in flight across these borders (TMA boxes in the 128-byte
// swizzle); four warps have 16 keys of each page:
//   scores, transposed:   S^T[16 keys x 8 rows] = K[16 x D] . Q^T,  keys as the 16-row operand of mma.m16n8k16, so that no row of it is padding
//   softmax over the keys: running maximum and sum per warp, base 2
//   O^T[D x 8 rows]     += V^T[D x 16 keys] . P^T
// bf16 pages come into the operands by ldmatrix.  Numbers of an 8-bit page are taken from shared memory in 16-byte pieces and become bf16 in registers: which
// component an element of an operand stands for is free as long as both operands agree, so the pieces of a thread are the components that its operand
// registers need, and the transposition of V costs no instruction beyond the byte permutation that spreads the numbers anyway.
// Partial results meet in chunk_merge_kernel, in the order of the runs.
// A row whose result is not a number, although its sum of weights is one, is worked out again over exactly its own keys (attend_row): a weight of zero times what a hidden key holds is no
// zero then.
#include "chunk_attn.cuh"
#include "tc_utils.cuh"
#include "mma_utils.cuh"
#include <math.h>
#include <algorithm>
#include <type_traits>

namespace jsm {

using namespace tc;

constexpr int CF_WARPS = 4;
constexpr int CF_THREADS = (CF_WARPS + 1) * 32;
constexpr float CF_NONE = -1.0e30f;  // the reference of a row that has seen nothing
constexpr float CF_RAISE = 8.0f;     // weights go up to 2^8 before the reference follows the maximum
constexpr int CF_ERR_FULL = 43, CF_ERR_EMPTY = 44;

__device__ __forceinline__ void cf_meet() { asm volatile("bar.sync 1, 128;" ::: "memory"); }  // the four warps that have keys
__device__ __forceinline__ uint32_t cf_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <int D, int NT, bool Q8>
struct FewSizes {
    static constexpr int ROWS = NT * 8;
    static constexpr int TILE = JSM_PAGE_SIZE * D * (Q8 ? 1 : 2);     // keys, or values, of a page
    static constexpr int STAGE = 2 * TILE + (Q8 ? 1024 : 0);          // keys | values | scales of both; bf16: for each 64 columns keys | values (1024-byte steps: the swizzle counts from there)
    static constexpr int STAGES = D == 128 && !Q8 ? 2 : 3;
    static constexpr int MEET = CF_WARPS * ROWS * D * 4;              // the warps' sums of a (sequence, kv head)
    static constexpr int SMEM = STAGES * STAGE + MEET + 1024;
    static constexpr int PER_SM = NT == 1 ? (Q8 ? 3 : 2) : 2;         // CTAs that share a multiprocessor
};

// The rows of a sequence are taken in groups of `per` tokens, each with the keys that it sees: for this kernel a group is a sequence of its own.
struct FewSeq {
    int row0, n_new, ctx;
};
// sequence s, if it has new tokens and no more rows than this kernel takes
template <bool EARLY = false>
__device__ __forceinline__ bool few_sequence(const ChunkArgs& a, const FewPlan& f, int s, FewSeq& q) { return chunk_lengths<EARLY>(a, s, q.row0, q.n_new, q.ctx) && q.n_new <= f.tokens; }
__device__ __forceinline__ FewSeq few_group(const FewPlan& f, const FewSeq& q, int group) {
    const int first = group * f.per, n = min(f.per, q.n_new - first);
    return FewSeq{q.row0 + first, n, q.ctx - q.n_new + first + n};
}
// pages that the queries of a group see, from page0 on
__device__ __forceinline__ int group_pages(const ChunkArgs& a, const FewSeq& q, int& page0) {
    page0 = first_key(a.window, q.ctx - q.n_new) / JSM_PAGE_SIZE;
    return (q.ctx - 1) / JSM_PAGE_SIZE + 1 - page0;
}
// all groups' of sequence s, for one kv head; 0: not this kernel's
template <bool EARLY = false>
__device__ __forceinline__ int head_pages(const ChunkArgs& a, const FewPlan& f, int s, FewSeq& q) {
    int sum = 0, page0;
    if (s < a.c.n_seqs && few_sequence<EARLY>(a, f, s, q))
        for (int g = 0; g * f.per < q.n_new; ++g) sum += group_pages(a, few_group(f, q, g), page0);
    return sum;
}
// Pages of a run, of the `all` pages of the call
__device__ __forceinline__ long long run_length(long long all, int n_runs) { return (all + n_runs - 1) / n_runs; }

template <int D, int NT, bool Q8>
__global__ void __launch_bounds__(CF_THREADS, FewSizes<D, NT, Q8>::PER_SM) chunk_few_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ CUtensorMap tmap_scales,
                                                                                            const __grid_constant__ ChunkArgs a, const __grid_constant__ FewPlan f, float* __restrict__ part) {
    using Z = FewSizes<D, NT, Q8>;
    constexpr int KS = D / 16;  // steps of 16 components; tiles of 16 components of O^T
    constexpr int few_rows = Z::ROWS;
    extern __shared__ uint8_t cf_dyn[];
    uint8_t* stages = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(cf_dyn) + 1023) & ~uintptr_t(1023));
    const uint32_t stages_u32 = smem_u32(stages);
    __shared__ uint64_t full_bar[Z::STAGES], empty_bar[Z::STAGES];
    __shared__ int abort_flag, sh_seq, sh_head, sh_group, sh_page, sh_pages;
    __shared__ FewSeq sh_q;
    __shared__ float sm_m[CF_WARPS][few_rows], sm_l[CF_WARPS][few_rows];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == CF_WARPS * 32) {
        for (int s = 0; s < Z::STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], CF_WARPS);
        }
        abort_flag = 0;
        mbar_fence_init();
    }
    chain_wait();
    chain_trigger();  // (now: the lengths that the merge reads before its own wait were written before this kernel's wait ended)
    if (warp == 0) {  // where this CTA's run begins
        long long all = 0;
        FewSeq q;
        for (int s0 = 0; s0 < a.c.n_seqs; s0 += 32) all += head_pages(a, f, s0 + lane, q);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        all *= a.c.Hkv;
        const long long len = run_length(all, gridDim.x), begin = blockIdx.x * len;
        if (lane == 0) sh_pages = (int)max(0ll, min(len, all - begin));
        long long before = 0;
        for (int s0 = 0; s0 < a.c.n_seqs && begin < all; s0 += 32) {
            const int n = head_pages(a, f, s0 + lane, q);
            long long sum = (long long)n * a.c.Hkv;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            const unsigned here = __ballot_sync(0xffffffffu, before + sum > begin);
            if (here) {
                if (lane == __ffs(here) - 1) {
                    const long long in = begin - (before + sum - (long long)n * a.c.Hkv);
                    sh_seq = s0 + lane;
                    sh_head = (int)(in / n);
                    int at = (int)(in % n), group = 0, page0;
                    for (int k = group_pages(a, few_group(f, q, 0), page0); at >= k; k = group_pages(a, few_group(f, q, group), page0)) {
                        at -= k;
                        ++group;
                    }
                    sh_group = group;
                    sh_page = at;
                    sh_q = q;
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
    }
    __syncthreads();
    int left = sh_pages, seq = sh_seq, hk = sh_head, group = sh_group, page = sh_page;
    if (left == 0) return;
    FewSeq whole_seq = sh_q, q = few_group(f, whole_seq, group);
    int page0, n_pages = group_pages(a, q, page0);
    // the next (sequence, kv head, group) of the run
    auto next = [&] {
        page = 0;
        if (++group * f.per >= whole_seq.n_new) {
            group = 0;
            if (++hk == a.c.Hkv) {
                hk = 0;
                do ++seq;
                while (!few_sequence(a, f, seq, whole_seq));
            }
        }
        q = few_group(f, whole_seq, group);
        n_pages = group_pages(a, q, page0);
    };

    if (warp == CF_WARPS) {
        if (lane == 0) {
            tma_prefetch_desc(&tmap);
            if (Q8) tma_prefetch_desc(&tmap_scales);
            int issued = 0;
            for (int s = 0, round = 0; issued < left; s = s + 1 == Z::STAGES ? (++round, 0) : s + 1) {
                if (round > 0 && !mbar_wait(&empty_bar[s], (round - 1) & 1, &abort_flag, a.c.err, CF_ERR_EMPTY)) break;
                const int id = cache_page(a.c, seq, (page0 + page) * JSM_PAGE_SIZE);
                uint8_t* dst = stages + s * Z::STAGE;
                // Keys and values of a page come by one request (a slab of 64 columns each, for bf16), the scales of both by another.  A page outside the pool: a place
                // before the first page, which reads as zeros.
                const int z = id < 0 ? -2 : 2 * id;
                mbar_expect_tx(&full_bar[s], 2 * Z::TILE + (Q8 ? 256 : 0));
                if constexpr (Q8) {
                    tma_load_3d(dst, &tmap, 0, hk * (JSM_PAGE_SIZE * D / 128), z, &full_bar[s]);
                    tma_load_3d(dst + 2 * Z::TILE, &tmap_scales, 0, hk, z, &full_bar[s]);
                } else {
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) tma_load_3d(dst + c * 16384, &tmap, c * 64, hk * JSM_PAGE_SIZE, z, &full_bar[s]);
                }
                if (++issued < left && ++page == n_pages) next();
            }
            if (abort_flag) {  // let the copies in flight land before the CTA exits (bounded)
                const long long t0 = clock64();
                for (int it = max(0, issued - Z::STAGES); it < issued; ++it)
                    while (!mbar_try_wait(&full_bar[it % Z::STAGES], (it / Z::STAGES) & 1) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
            }
        }
        return;
    }
    const int g = lane >> 2, t4 = lane & 3;
    const int mi = lane >> 3, mr = lane & 7;
    const int krow = warp * 16 + (mi & 1) * 8 + mr, kchunk = mi >> 1;   // ldmatrix, keys
    const int vrow = warp * 16 + (mi >> 1) * 8 + mr, vchunk = mi & 1;   // ldmatrix, values transposed
    // 8-bit pages: places of this lane's pieces in a stage (the keys of a warp are whole swizzle groups apart)
    uint32_t k_at[2], v_at[2][2];
    if constexpr (Q8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int byte = (warp * 16 + g + h * 8) * D + (D / 4) * t4, line = byte >> 7;
            k_at[h] = line * 128 + ((((byte >> 4) & 7) ^ (line & 7)) << 4);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int vb = (warp * 16 + t4 * 2 + h * 8 + i) * D + (D / 8) * g, vl = vb >> 7;
                v_at[h][i] = Z::TILE + vl * 128 + ((((vb >> 4) & 7) ^ (vl & 7)) << 4) + (D == 64 ? vb & 8 : 0);
            }
        }
    }
    float* sm_o = reinterpret_cast<float*>(stages + Z::STAGES * Z::STAGE);  // [warp][row][component], pairs of components where the lanes of a store meet different banks
    auto pair_at = [&](int w, int r, int p) {
        const int turn = (((r >> 1) & 3) << (Q8 && D == 64 ? 0 : 2)) ^ (Q8 && D == 128 ? (p >> 3) & 7 : 0);
        return sm_o + (w * few_rows + r) * D + (p ^ turn) * 2;
    };
    bool ok = true;
    int s = 0, round = 0;
    // B operand of the scores: row n * 8 + g, components of thread t4 in each step.  Of the next piece it is on its way while the sums of the one before meet.
    uint32_t qb[NT][KS][2];
    auto load_queries = [&] {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = n * 8 + g;
            const __nv_bfloat16* qp = a.q + (q.row0 + r / a.G) * a.q_rs + (long long)(hk * a.G + r % a.G) * D;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if constexpr (Q8) {
                    const uint2 w = r < q.n_new * a.G ? *reinterpret_cast<const uint2*>(qp + (D / 4) * t4 + 4 * ks) : make_uint2(0, 0);
                    qb[n][ks][0] = w.x;
                    qb[n][ks][1] = w.y;
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) qb[n][ks][h] = r < q.n_new * a.G ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + h * 8 + t4 * 2) : 0u;
                }
            }
        }
    };
    load_queries();
    for (bool first_piece = true;; first_piece = false) {  // a (sequence, kv head, group), or the run's piece of it
        const int row0 = q.row0, n_new = q.n_new, ctx = q.ctx, rows = n_new * a.G, lo = first_key(a.window, ctx - n_new);  // no row sees a key before it
        const int here = min(left, n_pages - page);
        const bool whole = here == n_pages;  // all of it: the result is final
        float m[NT][2], l[NT][2];  // rows (lane % 4) * 2 and + 1 of each tile
        float o[NT][KS][4];        // O^T
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = CF_NONE;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int j = 0; j < KS; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
        }
        int last[NT][2], first[NT][2];  // keys that the thread's two columns of each tile see
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int pos = ctx - n_new + min(n * 8 + t4 * 2 + h, rows - 1) / a.G;
                last[n][h] = pos;
                first[n][h] = first_key(a.window, pos);
            }
        }
        if constexpr (Q8) {  // components 0 and 2 of four, 1 and 3: the low bytes of a word of numbers, and the high ones
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint32_t x = qb[n][ks][0], y = qb[n][ks][1];
                    qb[n][ks][0] = __byte_perm(x, y, 0x5410);
                    qb[n][ks][1] = __byte_perm(x, y, 0x7632);
                }
        }
        const int all_from = first_key(a.window, ctx - 1), all_to = ctx - n_new;  // keys that every row sees
        // 16 keys of a page; MASKED: some of them are hidden from some row (the pages at both ends of what the sequence sees)
        auto step = [&](auto masked_tag, const uint32_t at, const int key0) {
            constexpr bool MASKED = decltype(masked_tag)::value;
            if (!Q8 && MASKED && (key0 < lo || key0 + 16 > ctx)) {  // values that no row sees: a weight of zero meets a number
                uint8_t* vb = stages + (at - stages_u32) + 8192;
                for (int i = lane; i < 16 * (D / 8); i += 32) {
                    const int row = warp * 16 + i / (D / 8), c = i % (D / 8), key = key0 + i / (D / 8);
                    if (key < lo || key >= ctx) *reinterpret_cast<uint4*>(vb + (c >> 3) * 16384 + row * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();  // the stage is overwritten by a bulk copy later
                __syncwarp();
            }
            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
            if constexpr (Q8) {
                uint32_t kw[2][D / 16];  // D / 4 numbers of keys g and g + 8
                uint32_t ks2[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    ks2[h] = lds16(at + 2 * Z::TILE + (warp * 16 + g + h * 8) * 2) * 0x00010001u;
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) {  // (the second piece of an even place is the next one, or the one before: bit 4 of the place)
                        const uint4 w = lds128(at + (k_at[h] ^ (c << 4)));
                        kw[h][c * 4] = w.x; kw[h][c * 4 + 1] = w.y; kw[h][c * 4 + 2] = w.z; kw[h][c * 4 + 3] = w.w;
                    }
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint32_t f[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        f[h] = q8_value2(kw[h][ks], ks2[h]);
                        f[h + 2] = q8_value2(kw[h][ks] >> 8, ks2[h]);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816(sc[n], f, qb[n][ks][0], qb[n][ks][1]);
                }
            } else {
                const uint32_t kbase = at;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const int c = ks * 2 + kchunk;
                    uint32_t f[4];
                    ldsm_x4(kbase + (c >> 3) * 16384 + krow * 128 + (((c & 7) ^ (krow & 7)) << 4), f);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816(sc[n], f, qb[n][ks][0], qb[n][ks][1]);
                }
            }
            // sc[n][0], [1]: key g, the thread's two rows; [2], [3]: key g + 8
            uint32_t pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = sc[n][i] * a.scale_log2;
                    if constexpr (MASKED) {
                        const int key = key0 + g + (i >> 1) * 8;
                        if (key < first[n][i & 1] || key > last[n][i & 1]) x[i] = -INFINITY;
                    }
                }
                // The reference follows the maximum only where a weight would pass 2^8: seldom after the first keys, so sums and accumulators are mostly left alone.
                if (__any_sync(0xffffffffu, fmaxf(x[0], x[2]) > m[n][0] + CF_RAISE || fmaxf(x[1], x[3]) > m[n][1] + CF_RAISE)) {
                    float corr[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float mx = fmaxf(x[h], x[h + 2]);
#pragma unroll
                        for (int sh = 4; sh < 32; sh <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, sh));
                        const float mn = fmaxf(m[n][h], mx);
                        corr[h] = fast_ex2(m[n][h] - mn);
                        m[n][h] = mn;
                        l[n][h] *= corr[h];
                    }
#pragma unroll
                    for (int j = 0; j < KS; ++j) {
                        o[n][j][0] *= corr[0];
                        o[n][j][1] *= corr[1];
                        o[n][j][2] *= corr[0];
                        o[n][j][3] *= corr[1];
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    x[h] = fast_ex2(x[h] - m[n][h]);
                    x[h + 2] = fast_ex2(x[h + 2] - m[n][h]);
                    l[n][h] += x[h] + x[h + 2];
                }
                pb[n][0] = cf_trans(pack_bf16x2(x[0], x[1]));
                pb[n][1] = cf_trans(pack_bf16x2(x[2], x[3]));
            }
            if constexpr (Q8) {
                uint32_t vw[4][D / 32], vs[2];  // D / 8 numbers of keys 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9: components (D / 8) g and up
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    vs[h] = lds32(at + 2 * Z::TILE + 128 + (warp * 16 + t4 * 2 + h * 8) * 2);
                    if constexpr (MASKED) {
                        const int key = key0 + t4 * 2 + h * 8;
                        if (key < lo || key >= ctx) vs[h] &= 0xFFFF0000u;
                        if (key + 1 < lo || key + 1 >= ctx) vs[h] &= 0x0000FFFFu;
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if constexpr (D == 128) {
                            const uint4 w = lds128(at + v_at[h][i]);
                            vw[h * 2 + i][0] = w.x; vw[h * 2 + i][1] = w.y; vw[h * 2 + i][2] = w.z; vw[h * 2 + i][3] = w.w;
                        } else {
                            const uint2 w = lds64(at + v_at[h][i]);
                            vw[h * 2 + i][0] = w.x; vw[h * 2 + i][1] = w.y;
                        }
                    }
                }
                // tile j: components (D / 8) g + 2 j (the tile's row g) and + 1 (its row g + 8)
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    uint32_t f[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t w0 = vw[h * 2][j >> 1], w1 = vw[h * 2 + 1][j >> 1];
                        f[h * 2] = q8_value2(__byte_perm(w0, w1, j & 1 ? 0x6622 : 0x4400), vs[h]);
                        f[h * 2 + 1] = q8_value2(__byte_perm(w0, w1, j & 1 ? 0x7733 : 0x5511), vs[h]);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816(o[n][j], f, pb[n][0], pb[n][1]);
                }
            } else {
                const uint32_t vbase = at + 8192;
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    const int c = j * 2 + vchunk;
                    uint32_t f[4];
                    ldsm_x4_trans(vbase + (c >> 3) * 16384 + vrow * 128 + (((c & 7) ^ (vrow & 7)) << 4), f);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816(o[n][j], f, pb[n][0], pb[n][1]);
                }
            }
        };
        for (int p = page; p < page + here; ++p) {
            ok = ok && mbar_wait_warp(&full_bar[s], round & 1, &abort_flag, a.c.err, CF_ERR_FULL);
            const int key0 = (page0 + p) * JSM_PAGE_SIZE + warp * 16;
            if (ok) {
                if (key0 >= all_from && key0 + 15 <= all_to) step(std::false_type{}, stages_u32 + s * Z::STAGE, key0);
                else if (key0 < ctx && key0 + 16 > lo) step(std::true_type{}, stages_u32 + s * Z::STAGE, key0);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty_bar[s]);
            if (++s == Z::STAGES) {
                s = 0;
                ++round;
            }
        }
        const int now_seq = seq, now_hk = hk;
        left -= here;
        if (left > 0) {
            next();
            load_queries();
        }
        // the four warps' sums meet (also after a wait that gave up: every warp comes by here as often)
        if (!first_piece) cf_meet();  // the piece before has been read
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int sh = 4; sh < 32; sh <<= 1) l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], sh);
                const int r = n * 8 + t4 * 2 + h;
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    if constexpr (Q8) {
                        *reinterpret_cast<float2*>(pair_at(warp, r, (D / 16) * g + j)) = make_float2(o[n][j][h], o[n][j][h + 2]);
                    } else {
                        pair_at(warp, r, j * 8 + (g >> 1))[g & 1] = o[n][j][h];
                        pair_at(warp, r, j * 8 + 4 + (g >> 1))[g & 1] = o[n][j][h + 2];
                    }
                }
                if (g == 0) {
                    sm_m[warp][r] = m[n][h];
                    sm_l[warp][r] = l[n][h];
                }
            }
        cf_meet();
        // a warp per row: the four warps' sums under their largest reference
        constexpr int N = D / 32;
        for (int r = warp; r < rows && !abort_flag; r += CF_WARPS) {
            float M = CF_NONE, L = 0.0f, acc[N];
#pragma unroll
            for (int w = 0; w < CF_WARPS; ++w) M = fmaxf(M, sm_m[w][r]);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < CF_WARPS; ++w) {
                const float f = fast_ex2(sm_m[w][r] - M);
                L += f * sm_l[w][r];
#pragma unroll
                for (int i = 0; i < N; i += 2) {
                    const float2 v = *reinterpret_cast<const float2*>(pair_at(w, r, lane * (N / 2) + i / 2));
                    acc[i] += f * v.x;
                    acc[i + 1] += f * v.y;
                }
            }
            const int row = row0 + r / a.G, head = now_hk * a.G + r % a.G;
            if (whole) {
                bool fine = true;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    acc[i] /= L;
                    fine = fine && fabsf(acc[i]) <= 3.402823466e38f;
                }
                if (__all_sync(0xffffffffu, fine || L != L)) {  // (a sum of weights that is a NaN: from a score of a key that the row sees)
                    __nv_bfloat16* dst = a.out + row * a.out_rs + (long long)head * D + lane * N;
#pragma unroll
                    for (int i = 0; i < N; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack_bf16x2(acc[i], acc[i + 1]);
                } else {
                    attend_row<D, Q8>(a, now_seq, row, head, ctx - n_new + r / a.G);
                }
            } else {
                // the run's first piece, or its last
                float* dst = part + ((blockIdx.x * 2ll + (first_piece ? 0 : 1)) * few_rows + r) * (D + 2);
#pragma unroll
                for (int i = 0; i < N; i += 2) *reinterpret_cast<float2*>(dst + lane * N + i) = make_float2(acc[i], acc[i + 1]);
                if (lane == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(M, L);
            }
        }
        if (left == 0) return;
    }
}

// The pieces of a row under their largest reference, in the order of the runs.  Few groups (JOIN): a block per (sequence, kv head, group) and row, each of four warps takes eight pieces
// of every 32, all their loads in flight, and they meet in shared memory.  Many groups, of a few pieces each: a warp per row (32 sequences of 8 tokens of 300, 32 heads: 32 us with the
// runs, a block per row 46).  What depends on the lengths alone is worked out while the runs are still under way: a kernel in front of the runs may have written them, but it has ended
// when the runs let this one start, so that they are in L2; L1 may still hold older ones (load_early).
constexpr int CM_RUNS = 8;
template <int D, bool Q8, bool JOIN>
__global__ void __launch_bounds__(128) chunk_merge_kernel(const __grid_constant__ ChunkArgs a, const __grid_constant__ FewPlan f, const float* part) {
    constexpr int N = D / 32, WARPS = JOIN ? 4 : 1;  // warps of a row
    __shared__ float sm_m[4], sm_l[4], sm_o[4][D];
    __shared__ long long sm_before[4], sm_all[4];
    const int most = gridDim.x / (a.c.n_seqs * a.c.Hkv), group = blockIdx.x % most, hk = blockIdx.x / most % a.c.Hkv, s = blockIdx.x / most / a.c.Hkv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = JOIN ? blockIdx.y : blockIdx.y * 4 + warp, few_rows = f.rows;
    long long before = 0, all = 0;
    FewSeq q = {0, 0, 0};
    for (int k = threadIdx.x; k < a.c.n_seqs; k += 128) {
        const int n = head_pages<true>(a, f, k, q);
        all += n;
        if (k < s) before += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        all += __shfl_xor_sync(0xffffffffu, all, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (lane == 0) {
        sm_all[warp] = all;
        sm_before[warp] = before;
    }
    int n_pages = 0, head_all = 0, groups_before = 0;
    if (few_sequence<true>(a, f, s, q))
        for (int g = 0, page0; g * f.per < q.n_new; ++g) {
            const int k = group_pages(a, few_group(f, q, g), page0);
            if (g < group) groups_before += k;
            if (g == group) n_pages = k;
            head_all += k;
        }
    __syncthreads();
    const long long len = max(1ll, run_length((sm_all[0] + sm_all[1] + sm_all[2] + sm_all[3]) * a.c.Hkv, f.n_runs));
    // the group's first page in the row of work
    const long long from = (sm_before[0] + sm_before[1] + sm_before[2] + sm_before[3]) * a.c.Hkv + (long long)hk * head_all + groups_before;
    const int c_first = (int)(from / len), n = n_pages > 0 ? (int)((from + n_pages - 1) / len) - c_first + 1 : 0;
    // the first piece of a run of its own, but for the first run, whose last piece it is unless it begins there
    const bool begins = from % len == 0;
    const int step = 2 * few_rows * (D + 2);
    const float* src = part + ((long long)c_first * 2 * few_rows + r) * (D + 2);
    auto piece = [&](int c) { return src + (long long)c * step + (c == 0 && !begins ? few_rows * (D + 2) : 0); };
    chain_wait();
    chain_trigger();
    if (n <= 1) return;
    q = few_group(f, q, group);
    if (r >= q.n_new * a.G) return;
    float m = CF_NONE, l = 0.0f, acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.0f;
    for (int c0 = JOIN ? warp * CM_RUNS : 0; c0 < n; c0 += WARPS * CM_RUNS) {
        float v[CM_RUNS][N];
        float2 ml = make_float2(CF_NONE, 0.0f);
        if (lane < CM_RUNS && c0 + lane < n) ml = *reinterpret_cast<const float2*>(piece(c0 + lane) + D);
#pragma unroll
        for (int c = 0; c < CM_RUNS; ++c) {
            const float* x = piece(min(c0 + c, n - 1)) + lane * N;
#pragma unroll
            for (int i = 0; i < N; i += 2) *reinterpret_cast<float2*>(&v[c][i]) = *reinterpret_cast<const float2*>(x + i);
        }
        const float mn = fmaxf(m, warp_max(ml.x)), corr = fast_ex2(m - mn);
        const float w0 = lane < CM_RUNS && c0 + lane < n ? fast_ex2(ml.x - mn) : 0.0f;
        m = mn;
        l = fmaf(l, corr, warp_sum(w0 * ml.y));
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] *= corr;
#pragma unroll
        for (int c = 0; c < CM_RUNS; ++c) {
            const float w = __shfl_sync(0xffffffffu, w0, c);
            if (c0 + c < n)
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] = fmaf(w, v[c][i], acc[i]);
        }
    }
    if constexpr (JOIN) {
        if (lane == 0) {
            sm_m[warp] = m;
            sm_l[warp] = l;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) sm_o[warp][lane * N + i] = acc[i];
        __syncthreads();
        if (warp != 0) return;
        m = CF_NONE;
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) m = fmaxf(m, sm_m[w]);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float x = fast_ex2(sm_m[w] - m);
            l += x * sm_l[w];
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] += x * sm_o[w][lane * N + i];
        }
    }
    bool fine = true;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        acc[i] /= l;
        fine = fine && fabsf(acc[i]) <= 3.402823466e38f;
    }
    const int t = q.row0 + r / a.G, head = hk * a.G + r % a.G;
    if (!__all_sync(0xffffffffu, fine || l != l)) {  // (as there)
        attend_row<D, Q8>(a, s, t, head, q.ctx - q.n_new + r / a.G);
        return;
    }
    __nv_bfloat16* dst = a.out + t * a.out_rs + (long long)head * D + lane * N;
#pragma unroll
    for (int i = 0; i < N; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack_bf16x2(acc[i], acc[i + 1]);
}

// As many runs as the chip holds CTAs (8-bit pages, heads of 128: three per multiprocessor with three stages each 80.7 us for 64 contexts of 512 to 8192, four with two 87.0; 77 by now), of
// two pages at least (one token over 4096 positions: 7.8 us, with runs of one page 8.1).
FewPlan chunk_few_plan(int n_seqs, int T, int max_new, int max_context, int Hkv, int G, int window, int rows, int tokens, int D, bool q8) {
    long long pages = ((long long)max_context + JSM_PAGE_SIZE - 1) / JSM_PAGE_SIZE;
    if (window > 0) pages = std::min(pages, ((long long)window + max_new + JSM_PAGE_SIZE - 3) / JSM_PAGE_SIZE + 1);
    FewPlan f;
    f.rows = rows;
    f.per = rows / G;
    f.tokens = std::min(tokens, max_new);
    const int per_sm = rows == 8 ? (q8 ? 3 : 2) : 2;
    const long long groups = std::min((long long)n_seqs * ((f.tokens + f.per - 1) / f.per), T / f.per + (long long)n_seqs);
    f.n_runs = (int)std::min((long long)per_sm * sm_count(), (pages * groups * Hkv + 1) / 2);
    f.merge = pages > 1;
    f.bytes = f.merge ? (size_t)f.n_runs * 2 * rows * (D + 2) * sizeof(float) : 0;
    return f;
}

template <int D, int NT, bool Q8>
static jsm_status few_go(const ChunkArgs& a, const FewPlan& f, float* part, cudaStream_t st) {
    using Z = FewSizes<D, NT, Q8>;
    // pool and scales as [keys or values of a page][kv heads x positions][D]
    CUtensorMap map, scales;
    const uint64_t Hkv = a.c.Hkv, halves = (uint64_t)a.c.n_pages * 2, lines = JSM_PAGE_SIZE * D / 128;
    jsm_status s = Q8 ? make_tmap_u8_3d(&map, a.c.pool, 128, Hkv * lines, halves, 128, Hkv * lines * 128, 128, lines, 2, true)
                      : make_tmap_bf16_3d(&map, a.c.pool, D, Hkv * JSM_PAGE_SIZE, halves, D, Hkv * JSM_PAGE_SIZE * D, 64, JSM_PAGE_SIZE, 2);
    if (s == JSM_OK && Q8) s = make_tmap_u8_3d(&scales, a.c.scales, 128, Hkv, halves, 128, Hkv * 128, 128, 1, 2, false);
    if (s != JSM_OK) return s;
    static DeviceOnce once;
    JSM_CUDA_CHECK(allow_shared(once, chunk_few_kernel<D, NT, Q8>, Z::SMEM));
    JSM_CUDA_CHECK(launch_chained(chunk_few_kernel<D, NT, Q8>, dim3(f.n_runs), dim3(CF_THREADS), (size_t)Z::SMEM, st, map, Q8 ? scales : map, a, f, part));
    JSM_LAUNCH_CHECK();
    if (f.merge) {
        const unsigned groups = (unsigned)a.c.n_seqs * a.c.Hkv * ((f.tokens + f.per - 1) / f.per), rows = (unsigned)std::min(f.per, f.tokens) * a.G;
        const bool join = groups * rows <= 8u * sm_count();
        const cudaError_t e = join ? launch_chained(chunk_merge_kernel<D, Q8, true>, dim3(groups, rows), dim3(128), 0, st, a, f, (const float*)part)
                                   : launch_chained(chunk_merge_kernel<D, Q8, false>, dim3(groups, (rows + 3) / 4), dim3(128), 0, st, a, f, (const float*)part);
        JSM_CUDA_CHECK(e);
        JSM_LAUNCH_CHECK();
    }
    return JSM_OK;
}

jsm_status chunk_few_launch(const ChunkArgs& a, const FewPlan& f, void* scratch, cudaStream_t st) {
    float* part = static_cast<float*>(scratch);
    if (a.c.D == 64) {
        if (a.c.scales) return f.rows == 8 ? few_go<64, 1, true>(a, f, part, st) : few_go<64, 2, true>(a, f, part, st);
        return f.rows == 8 ? few_go<64, 1, false>(a, f, part, st) : few_go<64, 2, false>(a, f, part, st);
    }
    if (a.c.scales) return f.rows == 8 ? few_go<128, 1, true>(a, f, part, st) : few_go<128, 2, true>(a, f, part, st);
    return f.rows == 8 ? few_go<128, 1, false>(a, f, part, st) : few_go<128, 2, false>(a, f, part, st);
}

}  // namespace jsm
