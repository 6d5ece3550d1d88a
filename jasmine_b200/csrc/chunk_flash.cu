// Attention of many new tokens of a sequence over its paged cache, bf16 or 8-bit, on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// The query rows of a kv head's group are one matrix, token after token, head after head within a token (row = token * G + head): a short portion of grouped
// queries fills the 128 rows of a tensor-core tile, and a key tile is fetched once for the whole group.  A CTA owns two such tiles of one (sequence, kv head)
// and walks the keys of its pages in tiles of 128 (two pages), as flash_attn.cu does: scores one key tile ahead of the products with V, the softmax of one
// query tile beside the tensor work of the other.
//   warp 0        copies: Q once (a box of tokens x heads x 64 components), key and value pages through rings
//   warp 1        issues the products: S_t = Q_t K^T, O_t += P_t V (P_t in TMEM over the first half of S_t)
//   warps 4-11    softmax, one thread per query row; register shares moved here from warps 0-3 (setmaxnreg)
//   warps 12-15   8-bit caches: numbers of a raw page -> bf16(n * scale) in the swizzled tiles that the tensor cores read.  Every number is exact in bf16 and every product
//                 rounded once, so scores and sums are those of a bf16 cache of these values; the conversion is spread over the whole group's rows
// Few tiles and long contexts: the CTAs of a cluster share the key tiles of one pair of query tiles; each sends the sums of the rows that another owns into that one's shared
// memory and joins its own with what it was sent, so that nothing goes through global memory and no second launch is needed.
// Values that no row of the CTA sees (behind the context, before the window) become zeros before they are multiplied; a row whose result is not a number is worked out
// again over exactly its own keys (attend_row).  Every wait is bounded.
#include "chunk_attn.cuh"
#include "tc_utils.cuh"
#include "softmax_rows.cuh"
#include "mma_utils.cuh"
#include <math.h>
#include <cmath>
#include <limits.h>
#include <stdlib.h>
#include <algorithm>
#include <mutex>
#include <type_traits>

namespace jsm {

using namespace tc;

constexpr int CK_BM = 128, CK_BN = 128;
constexpr int CK_SOFTMAX = 4, CK_CONVERT = 12;  // first warp of a role
constexpr float CK_RESCALE = 8.0f;             // the maximum is above the reference by so many powers of two: the reference follows
constexpr float CK_RAISE = 16777216.0f;        // a key tile's sum of weights is above 2^24: the reference is raised
constexpr float CK_NONE = -1.0e30f;             // the maximum of a row that has seen nothing

template <int D, bool Q8>
struct FlashSizes {
    static constexpr int THREADS = Q8 ? 512 : 384;
    static constexpr uint32_t SLAB = CK_BM * 64 * 2;                          // 64 columns of a tile
    static constexpr uint32_t TILE = D / 64 * SLAB;                           // 128 rows of Q, K or V
    static constexpr int ST = 2;
    static constexpr uint32_t RAW = Q8 ? JSM_PAGE_SIZE * D : 0;               // an 8-bit page of keys or values
    static constexpr uint32_t SMEM = (2 + 2 * ST) * TILE + 4 * RAW + 1024;    // Q | K ring | V ring | raw pages: keys 0, keys 1, values 0, values 1
};

struct FlashArgs {
    ChunkArgs a;
    int few_rows;      // sequences of so many rows are another kernel's
    int tile_tokens;   // tokens of a query tile
    int cluster;       // CTAs of a cluster
    int walk_tiles;    // key tiles that a CTA should walk at most: a sequence of more gives a pair of query tiles to 2, 4 .. CTAs of a cluster
    uint32_t inv_G;    // row / G = row * inv_G >> 16 for the rows of a tile
};

__device__ __forceinline__ void ck_cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void ck_cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t ck_peer(uint32_t local, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}
__device__ __forceinline__ void ck_store2(uint32_t addr, float a, float b) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}
__device__ __forceinline__ void ck_store4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// What a CTA is for: the cluster'th group of CTAs, of which it is number `rank`, serves so many pairs of query tiles of a sequence as the `share` CTAs of each leave room for; -1: none.
// For a whole warp.  The last tokens of a sequence, which see the most keys, come first for all heads: long CTAs do not start last (one prompt of 4096 tokens 158 us, with
// the pairs of a head next to one another 188).
struct Place {
    int seq, hk, tile, share, row0, n_new, ctx;
};
__device__ __forceinline__ Place find_tile(const FlashArgs& f, long long cluster, int rank) {
    const ChunkArgs& a = f.a;
    const int lane = threadIdx.x & 31, tokens = 2 * f.tile_tokens;
    Place p = {-1, 0, 0, 1, 0, 0, 0};
    for (int s0 = 0; s0 < a.c.n_seqs; s0 += 32) {
        const int s = s0 + lane;
        int n = 0, share = 1, row0 = 0, n_new = 0, ctx = 0;
        if (s < a.c.n_seqs && chunk_lengths(a, s, row0, n_new, ctx) && n_new * a.G > f.few_rows) {
            n = (n_new + tokens - 1) / tokens;
            const int keys = a.window > 0 ? min(ctx, a.window + tokens) : ctx;
            while (share < f.cluster && keys > f.walk_tiles * share * CK_BN) share *= 2;
        }
        const long long groups = ((long long)n * a.c.Hkv * share + f.cluster - 1) / f.cluster;
        long long sum = groups;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned here = __ballot_sync(0xffffffffu, sum > cluster);
        if (here) {
            const int w = __ffs(here) - 1, n_tiles = __shfl_sync(0xffffffffu, n, w);
            p.share = __shfl_sync(0xffffffffu, share, w);
            const long long in = (cluster - __shfl_sync(0xffffffffu, sum - groups, w)) * (f.cluster / p.share) + rank / p.share;
            p.row0 = __shfl_sync(0xffffffffu, row0, w);
            p.n_new = __shfl_sync(0xffffffffu, n_new, w);
            p.ctx = __shfl_sync(0xffffffffu, ctx, w);
            if (in < (long long)n_tiles * a.c.Hkv) {
                p.seq = s0 + w;
                p.hk = (int)(in % a.c.Hkv);
                p.tile = n_tiles - 1 - (int)(in / a.c.Hkv);
            }
            return p;
        }
        cluster -= __shfl_sync(0xffffffffu, sum, 31);
    }
    return p;
}

// What a CTA walks: query tile t has the tokens tok[t] and up (none: it is empty) and sees the key tiles jb[t] .. je[t]-1, counted from the page that holds the first key of the
// CTA's first token; the CTA's own are j_lo .. n_max-1.  No row sees a key before lo or from end on.
struct Walk {
    int tok[2], jb[2], je[2], lo, base, end, j_lo, n_max;
};
__device__ __forceinline__ Walk walk_of(const FlashArgs& f, const Place& p, int part) {
    Walk w;
    const int n_new = p.n_new, past = p.ctx - p.n_new, window = f.a.window;
    w.tok[0] = p.tile * 2 * f.tile_tokens;
    w.tok[1] = w.tok[0] + f.tile_tokens;
    w.lo = first_key(window, past + w.tok[0]);
    w.base = w.lo / JSM_PAGE_SIZE * JSM_PAGE_SIZE;
    w.end = past + min(w.tok[0] + 2 * f.tile_tokens, n_new);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        w.jb[t] = w.je[t] = 0;
        if (w.tok[t] < n_new) {
            w.jb[t] = (first_key(window, past + w.tok[t]) - w.base) / CK_BN;
            w.je[t] = (past + min(w.tok[t] + f.tile_tokens, n_new) - 1 - w.base) / CK_BN + 1;
        }
    }
    w.j_lo = w.jb[0];
    w.n_max = max(w.je[0], w.je[1]);
    if (p.share > 1) {  // this CTA's share of the key tiles
        const int len = (w.n_max - w.j_lo + p.share - 1) / p.share, from = w.j_lo + part * len, to = min(w.n_max, from + len);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            w.jb[t] = max(w.jb[t], from);
            w.je[t] = max(w.jb[t], min(w.je[t], to));
        }
        w.j_lo = min(from, to);
        w.n_max = to;
    }
    return w;
}

template <int D, bool Q8>
__global__ void __launch_bounds__(FlashSizes<D, Q8>::THREADS, 1)
    chunk_flash_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_kv, const __grid_constant__ FlashArgs f) {
    using Z = FlashSizes<D, Q8>;
    constexpr int ST = Z::ST;
    const ChunkArgs& a = f.a;
    extern __shared__ uint8_t ck_smem[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ck_smem) + 1023) & ~uintptr_t(1023));
    uint8_t* q_smem = tiles;
    uint8_t* k_smem = tiles + 2 * Z::TILE;
    uint8_t* v_smem = k_smem + ST * Z::TILE;
    uint8_t* raw_smem = v_smem + ST * Z::TILE;
    __shared__ __align__(8) uint64_t q_full, o_done;
    __shared__ __align__(8) uint64_t k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], raw_full[4], raw_empty[4];
    __shared__ __align__(8) uint64_t s_full[2], p_half[2], p_ready[2];
    __shared__ __align__(16) uint16_t raw_scales[4][JSM_PAGE_SIZE];
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_flag;
    __shared__ Place sh_place;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    chain_trigger();
    if (warp == 0 && elect_one()) {
        tma_prefetch_desc(&tmap_q);
        tma_prefetch_desc(&tmap_kv);
        abort_flag = 0;
        mbar_init(&q_full, 1);
        mbar_init(&o_done, 1);
        for (int s = 0; s < ST; ++s) {
            mbar_init(&k_full[s], Q8 ? 4 : 1);
            mbar_init(&v_full[s], Q8 ? 4 : 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        for (int s = 0; s < 4; ++s) { mbar_init(&raw_full[s], 1); mbar_init(&raw_empty[s], 4); }
        for (int t = 0; t < 2; ++t) { mbar_init(&s_full[t], 1); mbar_init(&p_half[t], 4); mbar_init(&p_ready[t], 4); }
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_smem, 512);
        tmem_relinquish();
    }
    chain_wait();
    const int rank = blockIdx.x % f.cluster;  // (clusters are consecutive blocks)
    int pages = 0;  // warp 0: pages of 16 key tiles at a time, lane i has the i-th
    auto load_pages = [&](int seq, const Walk& w, int j) {
        const int p = w.base / JSM_PAGE_SIZE + 2 * j + lane;
        return p * JSM_PAGE_SIZE < w.end ? cache_page(a.c, seq, p * JSM_PAGE_SIZE) : 0;
    };
    if (warp == 0) {
        __syncwarp();
        const Place p = find_tile(f, blockIdx.x / f.cluster, rank);
        if (lane == 0) sh_place = p;
        if (p.seq >= 0) {  // queries and the first pages are on their way before the block meets
            const Walk w = walk_of(f, p, rank % p.share);
            if (w.n_max > w.j_lo) {
                pages = load_pages(p.seq, w, w.j_lo);
                if (elect_one()) {
                    const int n_q = w.tok[1] < p.n_new ? 2 : 1;
                    mbar_expect_tx(&q_full, (uint32_t)(n_q * (D / 64) * f.tile_tokens * a.G) * 128);
                    for (int t = 0; t < n_q; ++t)
#pragma unroll
                        for (int c = 0; c < D / 64; ++c) tma_load_3d(q_smem + t * Z::TILE + c * Z::SLAB, &tmap_q, c * 64, p.hk * a.G, p.row0 + w.tok[t], &q_full);
                }
                __syncwarp();
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_smem;
    const uint32_t S_COL[2] = {0, 128}, O_COL[2] = {256, 256 + D};
    const int seq = sh_place.seq, hk = sh_place.hk, row0 = sh_place.row0, n_new = sh_place.n_new, ctx = sh_place.ctx, share = sh_place.share, part = rank % share;
    const bool work = seq >= 0;

    Walk w = {};
    if (work) w = walk_of(f, sh_place, part);
    const int past = ctx - n_new, lo = w.lo, base = w.base, end = w.end, j_lo = w.j_lo, n_max = w.n_max;
    const int(&tok)[2] = w.tok, (&jb)[2] = w.jb, (&je)[2] = w.je;

    if (warp < CK_SOFTMAX) regs_dec<Q8 ? 40 : 56>();
    if (warp == 0) {
        if (work && n_max > j_lo) {
            const int page0 = base / JSM_PAGE_SIZE, last_page = (end - 1) / JSM_PAGE_SIZE;  // (behind the context the last page again: hidden keys)
            int k_issued = 0, v_issued = 0;
            auto page_row = [&](int i, int half, int value) {  // row of the pool where the page of a key tile's half starts
                const int page = __shfl_sync(0xffffffffu, pages, (2 * i + half) & 31);
                return page < 0 ? -JSM_PAGE_SIZE : (int)cache_row(a.c, page, value, hk, 0);  // (outside the pool: rows before the first one, zeros)
            };
            for (int j = j_lo; j < n_max; ++j) {
                const int i = j - j_lo, s = i % ST;
                if ((i & 15) == 0 && i > 0) pages = load_pages(seq, w, j);
                int rows[2][2];
#pragma unroll
                for (int value = 0; value < 2; ++value)
#pragma unroll
                    for (int half = 0; half < 2; ++half) rows[value][half] = page_row(i, page0 + 2 * j + half <= last_page ? half : 0, value);
                if constexpr (Q8) {
                    bool ok = true;
#pragma unroll
                    for (int value = 0; value < 2; ++value)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const int slot = value * 2 + half, r = rows[value][half];
                            if (ok && i >= 1 && !mbar_wait_warp(&raw_empty[slot], (i & 1) ^ 1, &abort_flag, a.c.err, TC_TIMEOUT_EMPTY)) ok = false;
                            if (ok && elect_one()) {
                                mbar_expect_tx(&raw_full[slot], Z::RAW + (r < 0 ? 0 : 128));
                                tma_load_2d(raw_smem + slot * Z::RAW, &tmap_kv, 0, D == 64 ? r / 2 : r, &raw_full[slot]);  // (heads of 64: two positions in a line)
                                if (r >= 0) bulk_load(raw_scales[slot], a.c.scales + r, 128, &raw_full[slot]);
                            }
                            __syncwarp();
                            if (ok) k_issued = i * 4 + slot + 1;
                        }
                    if (!ok) break;
                } else {
                    if (i >= ST && !mbar_wait_warp(&k_empty[s], ((i / ST) & 1) ^ 1, &abort_flag, a.c.err, TC_TIMEOUT_EMPTY)) break;
                    if (elect_one()) {
                        mbar_expect_tx(&k_full[s], Z::TILE);
#pragma unroll
                        for (int c = 0; c < D / 64; ++c)
#pragma unroll
                            for (int half = 0; half < 2; ++half)
                                tma_load_2d(k_smem + s * Z::TILE + c * Z::SLAB + half * (Z::SLAB / 2), &tmap_kv, c * 64, rows[0][half], &k_full[s]);
                    }
                    __syncwarp();
                    k_issued = i + 1;
                    if (i >= ST && !mbar_wait_warp(&v_empty[s], ((i / ST) & 1) ^ 1, &abort_flag, a.c.err, TC_TIMEOUT_EMPTY)) break;
                    if (elect_one()) {
                        mbar_expect_tx(&v_full[s], Z::TILE);
#pragma unroll
                        for (int c = 0; c < D / 64; ++c)
#pragma unroll
                            for (int half = 0; half < 2; ++half)
                                tma_load_2d(v_smem + s * Z::TILE + c * Z::SLAB + half * (Z::SLAB / 2), &tmap_kv, c * 64, rows[1][half], &v_full[s]);
                    }
                    __syncwarp();
                    v_issued = i + 1;
                }
            }
            if (abort_flag) {  // let the copies in flight land before the CTA exits (bounded)
                const long long t0 = clock64();
                if constexpr (Q8) {
                    for (int i = max(0, k_issued - 4); i < k_issued; ++i)
                        while (!mbar_try_wait(&raw_full[i & 3], (i >> 2) & 1) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
                } else {
                    for (int i = max(0, k_issued - ST); i < k_issued; ++i)
                        while (!mbar_try_wait(&k_full[i % ST], (i / ST) & 1) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
                    for (int i = max(0, v_issued - ST); i < v_issued; ++i)
                        while (!mbar_try_wait(&v_full[i % ST], (i / ST) & 1) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
                }
                while (!mbar_try_wait(&q_full, 0) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
            }
        }
    } else if (warp == 1) {
        if (work && n_max > j_lo) {
            constexpr uint32_t idesc_qk = instr_desc_bf16(CK_BM, CK_BN, 0, 0), idesc_pv = instr_desc_bf16(CK_BM, D, 0, 1);
            bool ok = mbar_wait_warp(&q_full, 0, &abort_flag, a.c.err, TC_TIMEOUT_FULL);
            // S_t(j) = Q_t . K(j)^T over P_t(j - 1): the tensor pipe runs the products of this thread in order, the product with V has read P by then
            auto issue_s = [&](int t, uint32_t k_addr) {
                const uint32_t q_addr = smem_u32(q_smem + t * Z::TILE);
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = (kk / 4) * Z::SLAB;
                        mma_ss(tmem_base + S_COL[t], smem_desc_sw128(q_addr + off) + (uint64_t)((kk % 4) * 2), smem_desc_sw128(k_addr + off) + (uint64_t)((kk % 4) * 2),
                               idesc_qk, kk > 0 ? 1u : 0u);
                    }
                    mma_commit(&s_full[t]);
                }
                __syncwarp();
            };
            auto active = [&](int t, int j) { return j >= jb[t] && j < je[t]; };
            if (ok) {
                ok = mbar_wait_warp(&k_full[0], 0, &abort_flag, a.c.err, TC_TIMEOUT_FULL);
                tc_fence_after();
                if (ok) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        if (active(t, j_lo)) issue_s(t, smem_u32(k_smem));
                    if (elect_one()) mma_commit(&k_empty[0]);
                    __syncwarp();
                }
            }
            for (int j = j_lo; j < n_max && ok; ++j) {
                const int i = j - j_lo, vs = i % ST, s1 = (i + 1) % ST;
                const bool more = j + 1 < n_max;
                if (!mbar_wait_warp(&v_full[vs], (i / ST) & 1, &abort_flag, a.c.err, TC_TIMEOUT_FULL)) { ok = false; break; }
                if (!Q8) {  // values that no row sees: a weight of zero meets a number
                    const int key0 = base + j * CK_BN;
                    if (key0 < lo || key0 + CK_BN > end) {
                        uint8_t* vb = v_smem + vs * Z::TILE;
                        for (int n = lane; n < CK_BN * (D / 8); n += 32) {
                            const int row = n / (D / 8), c = n % (D / 8);
                            if (key0 + row < lo || key0 + row >= end)
                                *reinterpret_cast<uint4*>(vb + (c >> 3) * Z::SLAB + row * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                tc_fence_after();
                const uint32_t v_addr = smem_u32(v_smem + vs * Z::TILE), k_addr = smem_u32(k_smem + s1 * Z::TILE);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (active(t, j)) {
                        // The first half of the weights is taken while the second is being worked out: 2.24 -> 2.08 us per key tile.  (8-bit caches: 2.49 -> 2.55, so not there.)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            if ((half || !Q8) && !mbar_wait_warp(half ? &p_ready[t] : &p_half[t], (j - jb[t]) & 1, &abort_flag, a.c.err, TC_TIMEOUT_MISC)) { ok = false; break; }
                            tc_fence_after();
                            if ((half || !Q8) && elect_one()) {
#pragma unroll
                                for (int kk = Q8 ? 0 : half * 4; kk < half * 4 + 4; ++kk)
                                    mma_ts(tmem_base + O_COL[t], tmem_base + S_COL[t] + kk * 8, smem_desc_sw128_mn(v_addr + kk * 2048, Z::SLAB), idesc_pv,
                                           (j > jb[t] || kk > 0) ? 1u : 0u);
                            }
                            __syncwarp();
                        }
                        if (!ok) break;
                    }
                    if (t == 0 && more) {
                        if (!mbar_wait_warp(&k_full[s1], ((i + 1) / ST) & 1, &abort_flag, a.c.err, TC_TIMEOUT_FULL)) { ok = false; break; }
                        tc_fence_after();
                    }
                    if (active(t, j + 1)) issue_s(t, k_addr);
                }
                if (!ok) break;
                if (elect_one()) {
                    mma_commit(&v_empty[vs]);
                    if (more) mma_commit(&k_empty[s1]);
                }
                __syncwarp();
            }
            if (ok && elect_one()) mma_commit(&o_done);
            __syncwarp();
        }
    } else if (warp >= CK_SOFTMAX && warp < CK_CONVERT) {
        regs_inc<Q8 ? 200 : 224>();
        const int t = (warp - CK_SOFTMAX) / 4, quad = warp & 3, row = quad * 32 + lane;
        const int rows = f.tile_tokens * a.G;                       // rows of the tile that are queries
        const int token = tok[t] + (int)(row * f.inv_G >> 16), pos = past + token;   // (a row that is none has a position all the same)
        const bool query = work && row < rows && token < n_new;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quad * 32) << 16), s_addr = lane_addr + S_COL[t], o_addr = lane_addr + O_COL[t];
        const int pos_lo = past + tok[t], pos_hi = past + min(tok[t] + f.tile_tokens, n_new) - 1;  // first and last query of the tile
        // Weights are 2^(score - reference), whatever the reference: bf16, fp32 sums and fp32 accumulators keep their precision over 2^100 and more.  So the maximum is looked for
        // only where a row has no reference yet, or where keys are hidden; elsewhere a sum of weights above 2^24 raises the reference before the next key tile (a jump of
        // more than 2^100 within one tile gives infinities: such a row is worked out again at the end).
        float m_ref = query ? CK_NONE : 0.0f, l = 0.0f;
        int raise = 0;
        bool ok = true;
        auto rescale = [&](float alpha) {  // (TMEM accesses are the warp's: lanes whose reference stands use the factor 1)
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t r[32];
                tmem_ld32(o_addr + c, r);
                tmem_ld_wait();
                uint32_t w[16];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(__uint_as_float(r[half * 16 + i]) * alpha);
                    tmem_st16(o_addr + c + half * 16, w);
                }
            }
            l *= alpha;
        };
        for (int j = jb[t]; j < je[t] && ok; ++j) {
            if (!mbar_wait_warp(&s_full[t], (j - jb[t]) & 1, &abort_flag, a.c.err, TC_TIMEOUT_ACC)) { ok = false; break; }
            tc_fence_after();
            if (__any_sync(0xffffffffu, raise > 0)) {
                rescale(ex2_approx((float)-raise));
                m_ref += (float)raise;
            }
            uint32_t sr[CK_BN];
#pragma unroll
            for (int c = 0; c < CK_BN; c += 32) tmem_ld32(s_addr + c, reinterpret_cast<uint32_t(&)[32]>(sr[c]));
            tmem_ld_wait();
            float sv[CK_BN];
#pragma unroll
            for (int i = 0; i < CK_BN; ++i) sv[i] = __uint_as_float(sr[i]);
            const int key0 = base + j * CK_BN;
            const bool masked = key0 + CK_BN - 1 > pos_lo || key0 < first_key(a.window, pos_hi);
            if (__any_sync(0xffffffffu, masked || m_ref == CK_NONE)) {
                if (masked) {
                    const int from = first_key(a.window, pos) - key0, to = pos - key0;
#pragma unroll
                    for (int i = 0; i < CK_BN; ++i)
                        if (i < from || i > to) sv[i] = -INFINITY;
                }
                float mxs[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) mxs[k] = sv[k];
#pragma unroll
                for (int i = 8; i + 16 <= CK_BN; i += 16)
#pragma unroll
                    for (int k = 0; k < 8; ++k) mxs[k] = fmax3(mxs[k], sv[i + k], sv[i + 8 + k]);
#pragma unroll
                for (int k = 0; k < 8; ++k) mxs[k] = fmaxf(mxs[k], sv[CK_BN - 8 + k]);
                float mx = fmaxf(fmax3(mxs[0], mxs[1], mxs[2]), fmaxf(fmax3(mxs[3], mxs[4], mxs[5]), fmaxf(mxs[6], mxs[7])));
                mx *= a.scale_log2;
                const bool grow = mx > m_ref + CK_RESCALE;
                if (__any_sync(0xffffffffu, grow)) {
                    const float alpha = grow ? ex2_approx(m_ref - mx) : 1.0f;
                    if (j > jb[t]) rescale(alpha);
                    if (grow) m_ref = mx;
                }
            }
            // p = 2^(s - m_ref) as bf16 pairs over the first 64 columns of S.  All of them by the special-function unit: the warps are bound by issue here, a quarter by polynomials
            // on the FMA pipe costs 3 %.
            uint64_t ls2[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) ls2[k] = pack2(0.0f, 0.0f);
            const uint64_t neg_m2 = pack2(-m_ref, -m_ref), sc2 = pack2(a.scale_log2, a.scale_log2);
#pragma unroll
            for (int c = 0; c < CK_BN / 2; c += 16) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float x0, x1;
                    unpack2(ffma2(pack2(sv[2 * (c + i)], sv[2 * (c + i) + 1]), sc2, neg_m2), x0, x1);
                    const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
                    ls2[i & 3] = fadd2(ls2[i & 3], pack2(p0, p1));
                    w[i] = pack_bf16x2(p0, p1);
                }
                tmem_st16(s_addr + c, w);
                if (!Q8 && c == 16) {
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_half[t]);
                }
            }
            float la, lb;
            unpack2(fadd2(fadd2(ls2[0], ls2[1]), fadd2(ls2[2], ls2[3])), la, lb);
            const float sum = la + lb;
            l += sum;
            raise = sum > CK_RAISE ? (int)(__float_as_uint(sum) >> 23) - 127 : 0;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[t]);
        }
        if (ok && n_max > j_lo) ok = mbar_wait_warp(&o_done, 0, &abort_flag, a.c.err, TC_TIMEOUT_ACC);
        tc_fence_after();
        const bool any = ok && je[t] > jb[t];  // (the whole query tile)
        // What follows is executed once per CTA, mostly for the first time on its multiprocessor: rolled loops, because every line of code is fetched (unrolled, with the
        // factors of up to seven senders in registers, the end of a CTA took 4.2 us instead of 1.6).
        const int sw = warp - CK_SOFTMAX;
        // The meeting of a pair's CTAs, in place of tiles and rings: the rows of the eight softmax warps belong to the CTAs in equal shares; [sender][row of this CTA][D] sums and,
        // behind them, [sender][row] references and sums of the weights.
        const int own_rows = 2 * CK_BM / share;
        uint8_t* recv = tiles;
        uint8_t* recv_ml = tiles + (share - 1) * own_rows * (D * 4);
        uint8_t* staged = (share > 1 ? recv_ml + (share - 1) * own_rows * 8 : tiles) + sw * (32 * D * 2);  // this warp's 32 rows pass through here
        float own = 1.0f, L = l, M = m_ref;  // factor of the sums in TMEM, sum of the weights, reference of the row
        bool have = any;
        int senders = 0;
        const int warps = 8 / share, owner = sw / warps, r_own = sw % warps * 32;  // of a cluster: who joins this warp's rows, and where they are there
        auto sent_factor = [&](int p) {  // (0: that CTA had none of the row's keys)
            const float2 v = reinterpret_cast<const float2*>(recv_ml)[p * own_rows + r_own + lane];
            return make_float2(v.x == CK_NONE && v.y == 0.0f ? 0.0f : ex2_approx(v.x - M), v.y);
        };
        if (share > 1) {
            ck_cluster_arrive();
            ck_cluster_wait();  // every CTA has taken its products: tiles and rings may be overwritten
            if (owner != part) {
                const int at = (part < owner ? part : part - 1) * own_rows + r_own, peer = rank - part + owner;
                ck_store2(ck_peer(smem_u32(recv_ml) + (at + lane) * 8, peer), any ? m_ref : CK_NONE, any ? l : 0.0f);
                if (any) {
                    // a row per thread would send 16 bytes to 32 places at a time: through shared memory, so that eight lanes send 128 bytes
                    const uint32_t to = ck_peer(smem_u32(recv) + at * (D * 4), peer), here = smem_u32(staged);
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_addr + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 8; ++i) sts128(here + lane * 128 + ((i ^ (lane & 7)) * 16), make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const int r = k * 4 + (lane >> 3), piece = lane & 7;
                            const uint4 v = lds128(here + r * 128 + ((piece ^ (r & 7)) * 16));
                            ck_store4(to + r * (D * 4) + (((c / 4 + piece) ^ (r & 7)) * 16), v.x, v.y, v.z, v.w);
                        }
                        __syncwarp();
                    }
                }
            }
            ck_cluster_arrive();
            ck_cluster_wait();  // the sums are here
            have = owner == part && tok[t] < n_new;
            if (have) {
                senders = share - 1;
                if (!any) M = CK_NONE;
#pragma unroll 1
                for (int p = 0; p < senders; ++p) M = fmaxf(M, reinterpret_cast<const float2*>(recv_ml)[p * own_rows + r_own + lane].x);
                own = any ? ex2_approx(m_ref - M) : 0.0f;
                L = any ? l * own : 0.0f;
#pragma unroll 1
                for (int p = 0; p < senders; ++p) {
                    const float2 w = sent_factor(p);
                    if (w.x != 0.0f || w.y != 0.0f) L = fmaf(w.x, w.y, L);
                }
            }
        }
        if (have) {
            const float inv = 1.0f / L;
            bool bad = false;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float x[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = 0.0f;
                if (any) {
                    uint32_t r[32];
                    tmem_ld32(o_addr + c, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]) * own;
                }
#pragma unroll 2
                for (int p = 0; p < senders; ++p) {
                    const float w = sent_factor(p).x;
                    const uint8_t* src = recv + (p * own_rows + r_own + lane) * (D * 4);
                    if (w != 0.0f)
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 v = *reinterpret_cast<const float4*>(src + ((((c + i) / 4) ^ (lane & 7)) * 16));
                            x[i] = fmaf(w, v.x, x[i]);
                            x[i + 1] = fmaf(w, v.y, x[i + 1]);
                            x[i + 2] = fmaf(w, v.z, x[i + 2]);
                            x[i + 3] = fmaf(w, v.w, x[i + 3]);
                        }
                }
                float sum = 0.0f;  // (a component that is no number makes it one that is none either)
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    x[i] *= inv;
                    sum = fmaf(x[i], 0.0f, sum);
                }
                bad = bad || sum != 0.0f;
#pragma unroll
                for (int i = 0; i < 32; i += 8)
                    *reinterpret_cast<uint4*>(staged + lane * (D * 2) + ((((c + i) / 8) ^ (lane & 7)) * 16)) =
                        make_uint4(pack_bf16x2(x[i], x[i + 1]), pack_bf16x2(x[i + 2], x[i + 3]), pack_bf16x2(x[i + 4], x[i + 5]), pack_bf16x2(x[i + 6], x[i + 7]));
            }
            __syncwarp();
            // rows leave whole, 16 bytes per lane; lane r knows where row r goes
            constexpr int PIECES = D / 8, STEP = 32 / PIECES;
            const int piece = lane % PIECES, in = (int)(row * f.inv_G >> 16);
            const long long goes = query ? (row0 + token) * a.out_rs + (long long)(hk * a.G + row - in * a.G) * D : -1;
#pragma unroll 2
            for (int r0 = 0; r0 < 32; r0 += STEP) {
                const int r = r0 + lane / PIECES;
                const long long at = __shfl_sync(0xffffffffu, goes, r);
                const uint4 v = *reinterpret_cast<const uint4*>(staged + r * (D * 2) + ((piece ^ (r & 7)) * 16));
                if (at >= 0) *reinterpret_cast<uint4*>(a.out + at + piece * 8) = v;
            }
            __syncwarp();
            unsigned again = __ballot_sync(0xffffffffu, bad && query);
            while (again) {
                const int r = __ffs(again) - 1, at = quad * 32 + r, tk = tok[t] + at / a.G;
                again &= again - 1;
                attend_row<D, Q8>(a, seq, row0 + tk, hk * a.G + at % a.G, past + tk);
            }
        }
    } else if (Q8 && warp >= CK_CONVERT) {
        regs_dec<72>();
        if constexpr (Q8) {
            const int cw = warp - CK_CONVERT;
            // Reads and writes of 16 bytes, eight lanes at a time over all banks: the lanes have four pieces of two rows whose numbers differ in bit 0 (the places of the
            // bf16 pieces) and, where a row is a whole line, in bit 2 (the places of the raw pieces).  The loops over keys / values and the two pages stay rolled: unrolled,
            // the four warps wait for instructions (27 KB of them; 335 us for 1000 of 9000 positions).
            constexpr int STEPS = D == 128 ? 4 : 2;
            const int c4 = lane & 3, second = (lane >> 2) & 1;
            int row[STEPS];
            uint32_t src[STEPS], dst[STEPS];
#pragma unroll
            for (int n = 0; n < STEPS; ++n) {
                if constexpr (D == 128) {
                    const int slab = (lane >> 3) & 1, pair = (n & 1) * 2 + (lane >> 4), r = cw * 16 + (n >> 1) * 8 + (second ? pair ^ 5 : pair);
                    row[n] = r;
                    src[n] = r * 128 + (((slab * 4 + c4) ^ (r & 7)) << 4);
                    dst[n] = slab * Z::SLAB + r * 128 + (((c4 * 2) ^ (r & 7)) << 4);
                } else {
                    const int r = cw * 16 + n * 8 + (lane >> 3) * 2 + second, line = r >> 1;
                    row[n] = r;
                    src[n] = line * 128 + ((((r & 1) * 4 + c4) ^ (line & 7)) << 4);
                    dst[n] = r * 128 + (((c4 * 2) ^ (r & 7)) << 4);
                }
            }
            const uint32_t k_u32 = smem_u32(k_smem), v_u32 = smem_u32(v_smem), raw_sc = smem_u32(raw_scales);
            bool ok = true;
            for (int j = j_lo; j < n_max && ok; ++j) {
                const int i = j - j_lo, s = i % ST;
#pragma unroll 1
                for (int slot = 0; slot < 4; ++slot) {
                    const int value = slot >> 1, half = slot & 1;
                    if (half == 0 && i >= ST && !mbar_wait_warp(value ? &v_empty[s] : &k_empty[s], ((i / ST) & 1) ^ 1, &abort_flag, a.c.err, TC_TIMEOUT_EMPTY)) { ok = false; break; }
                    if (!mbar_wait_warp(&raw_full[slot], i & 1, &abort_flag, a.c.err, TC_TIMEOUT_FULL)) { ok = false; break; }
                    const uint32_t raw = smem_u32(raw_smem) + slot * Z::RAW;
                    const uint32_t to = (value ? v_u32 : k_u32) + s * Z::TILE + half * (JSM_PAGE_SIZE * 128);
                    // values that no row sees become zeros: a weight of zero meets a number
                    const int key0 = base + j * CK_BN + half * JSM_PAGE_SIZE, from = value ? lo - key0 : -1, until = value ? end - key0 : JSM_PAGE_SIZE;
                    uint4 w[STEPS];
                    uint32_t scale[STEPS];
#pragma unroll
                    for (int n = 0; n < STEPS; ++n) {
                        w[n] = lds128(raw + src[n]);
                        scale[n] = lds16(raw_sc + slot * (JSM_PAGE_SIZE * 2) + row[n] * 2);
                    }
#pragma unroll
                    for (int n = 0; n < STEPS; ++n) {
                        const uint32_t sc = row[n] < from || row[n] >= until ? 0u : scale[n] * 0x00010001u;
                        sts128(to + dst[n], make_uint4(q8_value2(__byte_perm(w[n].x, 0, 0x1100), sc), q8_value2(__byte_perm(w[n].x, 0, 0x3322), sc),
                                                       q8_value2(__byte_perm(w[n].y, 0, 0x1100), sc), q8_value2(__byte_perm(w[n].y, 0, 0x3322), sc)));
                        sts128(to + (dst[n] ^ 16), make_uint4(q8_value2(__byte_perm(w[n].z, 0, 0x1100), sc), q8_value2(__byte_perm(w[n].z, 0, 0x3322), sc),
                                                              q8_value2(__byte_perm(w[n].w, 0, 0x1100), sc), q8_value2(__byte_perm(w[n].w, 0, 0x3322), sc)));
                    }
                    if (half == 1) fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&raw_empty[slot]);
                        if (half == 1) mbar_arrive(value ? &v_full[s] : &k_full[s]);
                    }
                }
            }
        }
    }
    if (share > 1 && (warp < CK_SOFTMAX || warp >= CK_CONVERT)) {  // (the meeting counts every thread)
        ck_cluster_arrive();
        ck_cluster_wait();
        ck_cluster_arrive();
        ck_cluster_wait();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// clusters of S CTAs that the chip holds at once (15 of eight, 33 of four, although it has 148 multiprocessors)
template <int D, bool Q8>
static int flash_capacity(int S) {
    static std::mutex mu;
    static int known[64][9];  // per device
    int dev = -1;
    const int guess = S == 1 ? sm_count() : sm_count() / S * 3 / 4;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return guess;
    std::lock_guard<std::mutex> lock(mu);
    if (known[dev][S] == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(S * 256);
        cfg.blockDim = dim3(FlashSizes<D, Q8>::THREADS);
        cfg.dynamicSmemBytes = FlashSizes<D, Q8>::SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = S;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, chunk_flash_kernel<D, Q8>, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = guess;
        }
        known[dev][S] = n;
    }
    return known[dev][S];
}

template <int D, bool Q8>
static jsm_status flash_launch(const ChunkArgs& a, int few_rows, cudaStream_t st) {
    using Z = FlashSizes<D, Q8>;
    FlashArgs f{a, few_rows, CK_BM / a.G, 1, INT_MAX, (65536u + a.G - 1) / a.G};
    const long long tokens = 2ll * f.tile_tokens, per_seq = (a.max_new + tokens - 1) / tokens;
    const long long pairs = std::min(per_seq * a.c.n_seqs, a.T / tokens + a.c.n_seqs) * a.c.Hkv;  // at most
    static DeviceOnce once;
    JSM_CUDA_CHECK(allow_shared(once, chunk_flash_kernel<D, Q8>, (int)Z::SMEM));
    // CTAs of a pair of query tiles.  A key tile takes about 2 us, what is around the walk 6 us, a meeting 3 us: the longest CTA, or the chip's share of all and half a CTA's time
    // for the uneven end.  On average a pair of one sequence sees what lies before the middle of its new tokens, one of many sequences perhaps half of that.
    long long keys = a.max_context, mean = a.max_context - a.max_new / 2;
    if (a.c.n_seqs > 1) mean /= 2;
    if (a.window > 0) { keys = std::min(keys, (long long)a.window + tokens); mean = std::min(mean, keys); }
    const int key_tiles = (int)((keys + CK_BN - 1) / CK_BN);
    const float mean_tiles = (float)mean / CK_BN, likely = a.c.n_seqs > 1 ? (float)(a.T / tokens + a.c.n_seqs / 2 + 1) * a.c.Hkv : (float)pairs;
    float best = 0.0f;
    for (int S = 1; S <= 8; S *= 2) {
        if (S > 1 && key_tiles < 2 * S) break;
        const int cap = flash_capacity<D, Q8>(S) * S, walk = (key_tiles + S - 1) / S;
        const float around = 6.0f + (S > 1 ? 3.0f : 0.0f), longest = around + 2.0f * walk;
        const float ctas = likely * std::max(1.0f, mean_tiles / walk), one = around + 2.0f * std::min(mean_tiles, (float)walk);
        const float cost = ctas <= cap ? longest : std::max(longest, one * (ctas / cap + 0.5f));
        if (S == 1 || cost < best) { best = cost; f.cluster = S; f.walk_tiles = walk; }
    }
    if (pairs * f.cluster > INT32_MAX) JSM_FAIL(JSM_UNSUPPORTED, "jsm_attn_chunk: %lld tiles of queries", pairs);
    CUtensorMap mq, mkv;
    jsm_status s = make_tmap_bf16_3d(&mq, a.q, D, a.Hq, a.T, D, a.q_rs, 64, a.G, f.tile_tokens);
    if (s != JSM_OK) return s;
    const uint64_t rows = (uint64_t)a.c.n_pages * 2 * a.c.Hkv * JSM_PAGE_SIZE;
    s = Q8 ? make_tmap_u8_lines(&mkv, a.c.pool, rows * D / 128, JSM_PAGE_SIZE * D / 128) : make_tmap_bf16_2d(&mkv, a.c.pool, rows, D, D, JSM_PAGE_SIZE, 64);
    if (s != JSM_OK) return s;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(pairs * f.cluster));
    cfg.blockDim = dim3(Z::THREADS);
    cfg.dynamicSmemBytes = Z::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = f.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = chained_launch_enabled() ? attr : attr + 1;
    cfg.numAttrs = (chained_launch_enabled() ? 1 : 0) + (f.cluster > 1 ? 1 : 0);
    JSM_CUDA_CHECK(cudaLaunchKernelEx(&cfg, chunk_flash_kernel<D, Q8>, mq, mkv, f));
    JSM_LAUNCH_CHECK();
    return JSM_OK;
}

jsm_status chunk_flash_launch(const ChunkArgs& a, int few_rows, cudaStream_t st) {
    if (a.c.D == 64) return a.c.scales ? flash_launch<64, true>(a, few_rows, st) : flash_launch<64, false>(a, few_rows, st);
    return a.c.scales ? flash_launch<128, true>(a, few_rows, st) : flash_launch<128, false>(a, few_rows, st);
}

}  // namespace jsm
