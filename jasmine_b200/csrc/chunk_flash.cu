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
// 8-bit caches, long contexts (PAIR): two CTAs walk the keys of four query tiles together (cta_group::2).  A product has 256 rows, 128 in each CTA's tensor memory; each CTA brings and
// converts half of K (one page of two) and of V (64 of the 128 columns), so that a key tile is converted once for four query tiles, and operands come from shared memory half as
// often: 173 -> 148 us for 1000 tokens of 9000 positions (140 - 143 by now).  The even CTA issues the products of both; what the other has written is announced to it.  (bf16: 71 against 72 us for 512 of 8192,
// slower for prompts: without a conversion the hand-over between the CTAs costs what it saves.)
// Few tiles and long contexts: the units (CTAs or pairs) of a cluster share the key tiles of their query tiles; each sends the sums of the rows that another owns into that one's shared
// memory and joins its own with what it was sent, so that nothing goes through global memory and no second launch is needed.
// Values that no row of the CTA sees (behind the context, before the window) become zeros before they are multiplied; a row whose result is not a number, although its sum of weights is
// one, is worked out again over exactly its own keys (attend_row).  Every wait is bounded.
#include "chunk_attn.cuh"
#include "tc_utils.cuh"
#include "softmax_rows.cuh"
#include <math.h>
#include <limits.h>
#include <algorithm>
#include <mutex>
#include <type_traits>

namespace jsm {

using namespace tc;

constexpr int CK_BM = 128, CK_BN = 128;
constexpr int CK_SOFTMAX = 4, CK_CONVERT = 12;  // first warp of a role
constexpr float CK_RESCALE = 8.0f;             // the maximum is above the reference by so many powers of two: the reference follows
constexpr float CK_RAISE = 16777216.0f;        // a key tile's sum of weights is above 2^24: the reference is raised
constexpr float CK_JUMP = 1.3292279957849159e36f;  // ... above 2^120: the row is worked out again.  2^-120 is a factor that keeps its bits (below 2^-126 ex2_approx returns zero)
constexpr float CK_NONE = -1.0e30f;             // the maximum of a row that has seen nothing
constexpr float CK_AGAIN = -INFINITY;           // a row's sum of weights after such a jump

template <int D, bool Q8, bool PAIR>
struct FlashSizes {
    static constexpr int THREADS = Q8 ? 512 : 384;
    static constexpr uint32_t SLAB = CK_BM * 64 * 2;                          // 64 columns of a tile
    static constexpr uint32_t TILE = D / 64 * SLAB;                           // 128 rows of Q, K or V
    static constexpr uint32_t KV = PAIR ? TILE / 2 : TILE;                    // what the CTA has of a key tile's K (of a pair: a page) or V (half of the columns)
    static constexpr uint32_t K_SLAB = PAIR ? SLAB / 2 : SLAB;
    static constexpr int ST = PAIR ? 4 : 2;
    static constexpr int SLOTS = PAIR ? 3 : 4;                                // raw pages: keys (of a pair one page, else two), values 0, values 1
    static constexpr uint32_t RAW_K = JSM_PAGE_SIZE * D, RAW_V = PAIR ? RAW_K / 2 : RAW_K, RAW = Q8 ? (SLOTS - 2) * RAW_K + 2 * RAW_V : 0;
    static constexpr uint32_t SMEM = 2 * TILE + 2 * ST * KV + RAW + 1024;     // Q | K ring | V ring | raw pages
    static constexpr bool HALVES = PAIR || !Q8;                               // P is handed over in two halves
    static __device__ __forceinline__ uint32_t raw_at(int slot) { return PAIR && slot ? RAW_K + (slot - 1) * RAW_V : slot * RAW_K; }
    static_assert(!PAIR || (Q8 && D == 128));
};

struct FlashArgs {
    ChunkArgs a;
    int few_tokens;    // sequences of so many tokens are another kernel's
    int tile_tokens;   // tokens of a query tile
    int tiles;         // query tiles of a unit: a CTA's two, or a pair's four
    int cluster;       // units of a cluster
    int walk_tiles;    // key tiles that a CTA should walk at most: a sequence of more gives the query tiles of a unit to 2, 4 .. units of a cluster
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
// ---- pairs of CTAs (cta_group::2): the even CTA of a pair issues the products of both -------------------------------------
// Arrivals at a barrier of the other CTA (or this one), and waits for such.  What lies in tensor memory is ordered by tcgen05.wait and the tcgen05 fences on both sides; arrival and wait carry
// no more than the order of execution (relaxed, at the scope of the cluster).  What lies in shared memory, or is overwritten there behind the last products, needs a release and an acquire at
// that scope.  A thread pays for its release until all that it has written is there (by the converting warps 189 us for 1000 tokens of 9000 positions, by all arrivals 205), so the writers arrive in
// their own CTA, and one warp of the second CTA, which writes nothing itself, acquires that and releases it to the first: 143 us (139 with arrivals that release to their own CTA only, an order
// that the memory model does not give).
__device__ __forceinline__ void ck_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void ck_arrive_tmem(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
template <bool TMEM>
__device__ __forceinline__ bool ck_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t d;
    if constexpr (TMEM)
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(d) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    else
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(d) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return d != 0;
}
// mbar_wait_warp for a barrier at which the other CTA of a pair, or its products, arrive too
template <bool PAIR, bool TMEM = false>
__device__ __forceinline__ bool ck_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
    if constexpr (!PAIR) return mbar_wait_warp(bar, parity, abort_flag, err, code);
    bool ok = ck_try_wait<TMEM>(bar, parity);
    for (const long long t0 = ok ? 0 : clock64(); !ok;) {
        ok = ck_try_wait<TMEM>(bar, parity);
        if (ok || *abort_flag) break;
        if (clock64() - t0 > WAIT_LIMIT_CYCLES) {
            *abort_flag = 1;
            if (err) atomicCAS(err, 0, code);
            break;
        }
    }
    return __all_sync(0xffffffffu, ok);
}
template <bool PAIR>
__device__ __forceinline__ void ck_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else mma_ss(d, a, b, idesc, accumulate);
}
template <bool PAIR>
__device__ __forceinline__ void ck_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else mma_ts(d, a, b, idesc, accumulate);
}
// arrives at `bar` (of a pair: in both CTAs) once the products issued so far are done
template <bool PAIR>
__device__ __forceinline__ void ck_commit(uint64_t* bar, uint32_t pair_mask) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)pair_mask) : "memory");
    else mma_commit(bar);
}
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// What a unit (a CTA, or a pair) is for: the cluster'th group of units, of which it is number `rank`, serves so many units' query tiles of a sequence as the `share` units of each leave
// room for; -1: none.
// For a whole warp.  The last tokens of a sequence, which see the most keys, come first for all heads: long CTAs do not start last (one prompt of 4096 tokens 158 us, with
// the pairs of a head next to one another 188).
struct Place {
    int seq, hk, tile, share, row0, n_new, ctx;
};
__device__ __forceinline__ Place find_tile(const FlashArgs& f, long long cluster, int rank) {
    const ChunkArgs& a = f.a;
    const int lane = threadIdx.x & 31, tokens = f.tiles * f.tile_tokens;
    Place p = {-1, 0, 0, 1, 0, 0, 0};
    for (int s0 = 0; s0 < a.c.n_seqs; s0 += 32) {
        const int s = s0 + lane;
        int n = 0, share = 1, row0 = 0, n_new = 0, ctx = 0;
        if (s < a.c.n_seqs && chunk_lengths(a, s, row0, n_new, ctx) && n_new > f.few_tokens) {
            n = (n_new + tokens - 1) / tokens;
            const int keys = a.window > 0 ? (int)min((long long)ctx, (long long)a.window + tokens) : ctx;
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

// What a CTA walks: its query tile t has the tokens tok[t] and up (none: it is empty) and meets the key tiles jb[t] .. je[t]-1, those that it sees or its pair's other tile t does, counted
// from the page that holds the first key of the unit's first token; the unit's own are j_lo .. n_max-1.  No row sees a key before lo or from end on.
struct Walk {
    int tok[2], jb[2], je[2], lo, base, end, j_lo, n_max;
};
__device__ __forceinline__ Walk walk_of(const FlashArgs& f, const Place& p, int part, int side) {
    Walk w;
    const int n_new = p.n_new, past = p.ctx - p.n_new, window = f.a.window, tok0 = p.tile * f.tiles * f.tile_tokens, both = f.tiles / 2 * f.tile_tokens;
    w.lo = first_key(window, past + tok0);
    w.base = w.lo / JSM_PAGE_SIZE * JSM_PAGE_SIZE;
    w.end = past + min(tok0 + 2 * both, n_new);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int first = tok0 + t * both;
        w.tok[t] = first + side * f.tile_tokens;
        w.jb[t] = w.je[t] = 0;
        if (first < n_new) {
            w.jb[t] = (first_key(window, past + first) - w.base) / CK_BN;
            w.je[t] = (past + min(first + both, n_new) - 1 - w.base) / CK_BN + 1;
        }
    }
    w.j_lo = w.jb[0];
    w.n_max = max(w.je[0], w.je[1]);
    if (p.share > 1) {  // this unit's share of the key tiles
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

template <int D, bool Q8, bool PAIR>
__global__ void __launch_bounds__(FlashSizes<D, Q8, PAIR>::THREADS, 1)
    chunk_flash_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_kv, const __grid_constant__ CUtensorMap tmap_half, const __grid_constant__ FlashArgs f) {
    using Z = FlashSizes<D, Q8, PAIR>;
    constexpr int ST = Z::ST;
    const ChunkArgs& a = f.a;
    extern __shared__ uint8_t ck_smem[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ck_smem) + 1023) & ~uintptr_t(1023));
    uint8_t* q_smem = tiles;
    uint8_t* k_smem = tiles + 2 * Z::TILE;
    uint8_t* v_smem = k_smem + ST * Z::KV;
    uint8_t* raw_smem = v_smem + ST * Z::KV;
    __shared__ __align__(8) uint64_t q_full, o_done;
    __shared__ __align__(8) uint64_t k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], raw_full[4], raw_empty[4];
    __shared__ __align__(8) uint64_t s_full[2], p_half[2], p_ready[2];
    __shared__ __align__(16) uint16_t raw_scales[4][JSM_PAGE_SIZE];
    __shared__ uint32_t tmem_base_smem;
    __shared__ int abort_flag;
    __shared__ Place sh_place;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ctas = PAIR ? 2 * f.cluster : f.cluster, rank = blockIdx.x % ctas;  // (clusters are consecutive blocks)
    const int side = PAIR ? rank & 1 : 0, unit = PAIR ? rank >> 1 : rank;
    const bool leads = side == 0;
    chain_trigger();
    if (warp == 0 && elect_one()) {
        tma_prefetch_desc(&tmap_q);
        tma_prefetch_desc(&tmap_kv);
        abort_flag = 0;
        // the leader of a pair hears of the other CTA's queries and converted pages from that one's warp 1, of its weights from the warps that write them
        const int both = PAIR && leads ? 2 : 1;
        mbar_init(&q_full, both);
        mbar_init(&o_done, 1);
        for (int s = 0; s < ST; ++s) {
            mbar_init(&k_full[s], Q8 ? 3 + both : both);
            mbar_init(&v_full[s], Q8 ? 3 + both : both);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        for (int s = 0; s < 4; ++s) { mbar_init(&raw_full[s], 1); mbar_init(&raw_empty[s], 4); }
        for (int t = 0; t < 2; ++t) { mbar_init(&s_full[t], 1); mbar_init(&p_half[t], 4 * both); mbar_init(&p_ready[t], 4 * both); }
        mbar_fence_init();
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_smem)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            tmem_alloc(&tmem_base_smem, 512);
            tmem_relinquish();
        }
    }
    chain_wait();
    int pages = 0;  // warp 0: pages of 16 key tiles at a time, lane i has the i-th
    auto load_pages = [&](int seq, const Walk& w, int j) {
        const int p = w.base / JSM_PAGE_SIZE + 2 * j + lane;
        return p <= (w.end - 1) / JSM_PAGE_SIZE ? cache_page(a.c, seq, p * JSM_PAGE_SIZE) : 0;  // (pages: the place of a key behind the context may pass 32 bits)
    };
    if (warp == 0) {
        __syncwarp();
        const Place p = find_tile(f, blockIdx.x / ctas, unit);
        if (lane == 0) sh_place = p;
        if (p.seq >= 0) {  // queries and the first pages are on their way before the block meets
            const Walk w = walk_of(f, p, unit % p.share, side);
            if (w.n_max > w.j_lo) {
                pages = load_pages(p.seq, w, w.j_lo);
                if (elect_one()) {
                    const int n_q = w.tok[1] < p.n_new ? 2 : w.tok[0] < p.n_new ? 1 : 0;
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
    if (PAIR) {
        ck_cluster_arrive();
        ck_cluster_wait();  // both CTAs' barriers and tensor memory exist
    }
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_smem;
    const uint32_t S_COL[2] = {0, 128}, O_COL[2] = {256, 256 + D};
    const int seq = sh_place.seq, hk = sh_place.hk, row0 = sh_place.row0, n_new = sh_place.n_new, ctx = sh_place.ctx, share = sh_place.share, part = unit % share;
    const bool work = seq >= 0;

    Walk w = {};
    if (work) w = walk_of(f, sh_place, part, side);
    const int past = ctx - n_new, lo = w.lo, base = w.base, end = w.end, j_lo = w.j_lo, n_max = w.n_max;
    const int(&tok)[2] = w.tok, (&jb)[2] = w.jb, (&je)[2] = w.je;

    if (warp < CK_SOFTMAX) regs_dec<Q8 ? 56 : 72>();
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
                            if (PAIR && !value && half) continue;  // (keys: one page)
                            const int slot = PAIR ? value + half : value * 2 + half, r = PAIR && !value && side ? rows[0][1] : rows[value][half];
                            if (ok && i >= 1 && !mbar_wait_warp(&raw_empty[slot], (i & 1) ^ 1, &abort_flag, a.c.err, TC_TIMEOUT_EMPTY)) ok = false;
                            if (ok && elect_one()) {
                                mbar_expect_tx(&raw_full[slot], (value ? Z::RAW_V : Z::RAW_K) + (r < 0 ? 0 : 128));
                                if (PAIR && value) tma_load_2d(raw_smem + Z::raw_at(slot), &tmap_half, side * 64, r, &raw_full[slot]);
                                else tma_load_2d(raw_smem + Z::raw_at(slot), &tmap_kv, 0, D == 64 ? r / 2 : r, &raw_full[slot]);  // (heads of 64: two positions in a line)
                                if (r >= 0) bulk_load(raw_scales[slot], a.c.scales + r, 128, &raw_full[slot]);
                            }
                            __syncwarp();
                            if (ok) k_issued = i * Z::SLOTS + slot + 1;
                        }
                    if (!ok) break;
                } else {
                    if (i >= ST && !mbar_wait_warp(&k_empty[s], ((i / ST) & 1) ^ 1, &abort_flag, a.c.err, TC_TIMEOUT_EMPTY)) break;
                    if (elect_one()) {
                        mbar_expect_tx(&k_full[s], Z::KV);
#pragma unroll
                        for (int c = 0; c < D / 64; ++c)
#pragma unroll
                            for (int half = 0; half < 2; ++half)
                                tma_load_2d(k_smem + s * Z::KV + c * Z::SLAB + half * (Z::SLAB / 2), &tmap_kv, c * 64, rows[0][half], &k_full[s]);
                    }
                    __syncwarp();
                    k_issued = i + 1;
                    if (i >= ST && !mbar_wait_warp(&v_empty[s], ((i / ST) & 1) ^ 1, &abort_flag, a.c.err, TC_TIMEOUT_EMPTY)) break;
                    if (elect_one()) {
                        mbar_expect_tx(&v_full[s], Z::KV);
#pragma unroll
                        for (int c = 0; c < D / 64; ++c)
#pragma unroll
                            for (int half = 0; half < 2; ++half)
                                tma_load_2d(v_smem + s * Z::KV + c * Z::SLAB + half * (Z::SLAB / 2), &tmap_kv, c * 64, rows[1][half], &v_full[s]);
                    }
                    __syncwarp();
                    v_issued = i + 1;
                }
            }
            if (abort_flag) {  // let the copies in flight land before the CTA exits (bounded)
                const long long t0 = clock64();
                if constexpr (Q8) {
                    for (int i = max(0, k_issued - Z::SLOTS); i < k_issued; ++i)
                        while (!mbar_try_wait(&raw_full[i % Z::SLOTS], (i / Z::SLOTS) & 1) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
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
        if (PAIR && work && n_max > j_lo && !leads) {  // the leader hears that the other CTA's queries, keys and values are there
            const uint32_t q_to = ck_peer(smem_u32(&q_full), rank - 1), k_to = ck_peer(smem_u32(k_full), rank - 1), v_to = ck_peer(smem_u32(v_full), rank - 1);
            bool ok = mbar_wait_warp(&q_full, 0, &abort_flag, a.c.err, TC_TIMEOUT_FULL);
            if (ok && lane == 0) ck_arrive(q_to);
            for (int j = j_lo; j < n_max && ok; ++j) {
                const int i = j - j_lo, s = i % ST;
                ok = mbar_wait_warp(&k_full[s], (i / ST) & 1, &abort_flag, a.c.err, TC_TIMEOUT_FULL);
                if (ok && lane == 0) ck_arrive(k_to + s * 8);
                ok = ok && mbar_wait_warp(&v_full[s], (i / ST) & 1, &abort_flag, a.c.err, TC_TIMEOUT_FULL);
                if (ok && lane == 0) ck_arrive(v_to + s * 8);
            }
        }
        if (work && n_max > j_lo && leads) {
            constexpr uint32_t idesc_qk = instr_desc_bf16(PAIR ? 2 * CK_BM : CK_BM, CK_BN, 0, 0), idesc_pv = instr_desc_bf16(PAIR ? 2 * CK_BM : CK_BM, D, 0, 1);
            const uint32_t pair_mask = 3u << rank;
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                return ck_wait_warp<PAIR>(bar, parity, &abort_flag, a.c.err, code);
            };
            bool ok = wait(&q_full, 0, TC_TIMEOUT_FULL);
            // S_t(j) = Q_t . K(j)^T over P_t(j - 1): the tensor pipe runs the products of this thread in order, the product with V has read P by then
            uint64_t q_desc[2] = {smem_desc_sw128(smem_u32(q_smem)), smem_desc_sw128(smem_u32(q_smem + Z::TILE))};
            auto ready = [](uint64_t& desc) { asm volatile("" : "+l"(desc)); };  // (worked out here, not behind a wait)
            ready(q_desc[0]);
            ready(q_desc[1]);
            auto issue_s = [&](int t, uint64_t k_desc) {
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        ck_mma_ss<PAIR>(tmem_base + S_COL[t], q_desc[t] + (uint64_t)((kk / 4) * (Z::SLAB >> 4) + (kk % 4) * 2), k_desc + (uint64_t)((kk / 4) * (Z::K_SLAB >> 4) + (kk % 4) * 2), idesc_qk, kk > 0 ? 1u : 0u);
                    }
                    ck_commit<PAIR>(&s_full[t], pair_mask);
                }
                __syncwarp();
            };
            auto active = [&](int t, int j) { return j >= jb[t] && j < je[t]; };
            if (ok) {
                ok = wait(&k_full[0], 0, TC_TIMEOUT_FULL);
                tc_fence_after();
                if (ok) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        if (active(t, j_lo)) issue_s(t, smem_desc_sw128(smem_u32(k_smem)));
                    if (elect_one()) ck_commit<PAIR>(&k_empty[0], pair_mask);
                    __syncwarp();
                }
            }
            for (int j = j_lo; j < n_max && ok; ++j) {
                const int i = j - j_lo, vs = i % ST, s1 = (i + 1) % ST;
                const bool more = j + 1 < n_max;
                // (the next keys too: nothing but the products themselves is to come between the weights' arrival and the next scores)
                if (!wait(&v_full[vs], (i / ST) & 1, TC_TIMEOUT_FULL) || (more && !wait(&k_full[s1], ((i + 1) / ST) & 1, TC_TIMEOUT_FULL))) { ok = false; break; }
                if (!Q8) {  // values that no row sees: a weight of zero meets a number
                    const int key0 = base + j * CK_BN;
                    if (key0 < lo || end - key0 < CK_BN) {
                        uint8_t* vb = v_smem + vs * Z::KV;
                        for (int n = lane; n < CK_BN * (D / 8); n += 32) {
                            const int row = n / (D / 8), c = n % (D / 8);
                            if (key0 + row < lo || row >= end - key0)
                                *reinterpret_cast<uint4*>(vb + (c >> 3) * Z::SLAB + row * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                tc_fence_after();
                uint64_t v_desc = smem_desc_sw128_mn(smem_u32(v_smem + vs * Z::KV), Z::SLAB), k_desc = smem_desc_sw128(smem_u32(k_smem + s1 * Z::KV));
                ready(v_desc);
                ready(k_desc);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (active(t, j)) {
                        // The first half of the weights is taken while the second is being worked out: 2.24 -> 2.08 us per key tile.  (8-bit caches: 2.49 -> 2.55 of a CTA
                        // alone, whose converting warps are behind, so not there; pairs 2.13 -> 2.10.)
                        constexpr int N = Z::HALVES ? 2 : 1, BLOCKS = CK_BN / 16 / N;
#pragma unroll
                        for (int half = 0; half < N; ++half) {
                            if (!wait(half == N - 1 ? &p_ready[t] : &p_half[t], (j - jb[t]) & 1, TC_TIMEOUT_MISC)) { ok = false; break; }
                            tc_fence_after();
                            if (elect_one()) {
#pragma unroll
                                for (int kk = half * BLOCKS; kk < (half + 1) * BLOCKS; ++kk)
                                    ck_mma_ts<PAIR>(tmem_base + O_COL[t], tmem_base + S_COL[t] + kk * 8, v_desc + (uint64_t)(kk * (2048 >> 4)), idesc_pv,
                                                    (j > jb[t] || kk > 0) ? 1u : 0u);
                            }
                            __syncwarp();
                        }
                        if (!ok) break;
                    }
                    if (active(t, j + 1)) issue_s(t, k_desc);
                }
                if (!ok) break;
                if (elect_one()) {
                    ck_commit<PAIR>(&v_empty[vs], pair_mask);
                    if (more) ck_commit<PAIR>(&k_empty[s1], pair_mask);
                }
                __syncwarp();
            }
            if (ok && elect_one()) ck_commit<PAIR>(&o_done, pair_mask);
            __syncwarp();
        }
    } else if (warp >= CK_SOFTMAX && warp < CK_CONVERT) {
        regs_inc<Q8 ? 192 : 216>();  // (200 and 40 for the first four warps: those spill, 152 us instead of 148 for 1000 tokens of 9000 positions of an 8-bit cache)
        const int t = (warp - CK_SOFTMAX) / 4, quad = warp & 3, row = quad * 32 + lane;
        const int rows = f.tile_tokens * a.G;                       // rows of the tile that are queries
        const int token = tok[t] + (int)(row * f.inv_G >> 16), pos = past + token;   // (a row that is none has a position all the same)
        const bool query = work && row < rows && token < n_new;
        const uint32_t lane_addr = tmem_base + ((uint32_t)(quad * 32) << 16), s_addr = lane_addr + S_COL[t], o_addr = lane_addr + O_COL[t];
        const int pos_lo = past + tok[t], pos_hi = past + min(tok[t] + f.tile_tokens, n_new) - 1;  // first and last query of the tile
        // Weights are 2^(score - reference), whatever the reference: bf16, fp32 sums and fp32 accumulators keep their precision over 2^100 and more.  So the maximum is looked for
        // only where a row has no reference yet, or where keys are hidden; elsewhere a sum of weights above 2^24 raises the reference before the next key tile, or behind the last.  A
        // key tile's sum above 2^120, or one that is infinite, marks the row's sum of weights for good: such a row is worked out again at the end.
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
            if (l != CK_AGAIN) l *= alpha;
        };
        const bool mine = tok[t] < n_new;  // (of a pair the other CTA may have a tile alone)
        const uint32_t half_to = PAIR ? ck_peer(smem_u32(&p_half[t]), rank & ~1) : 0, ready_to = PAIR ? ck_peer(smem_u32(&p_ready[t]), rank & ~1) : 0;
        auto weights_are_there = [&](uint64_t* bar, uint32_t to) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) ck_arrive_tmem(to);
                else mbar_arrive(bar);
            }
        };
        for (int j = jb[t]; j < je[t] && ok; ++j) {
            if (!ck_wait_warp<PAIR, true>(&s_full[t], (j - jb[t]) & 1, &abort_flag, a.c.err, TC_TIMEOUT_ACC)) { ok = false; break; }
            tc_fence_after();
            if (PAIR && !mine) {
                weights_are_there(&p_half[t], half_to);
                weights_are_there(&p_ready[t], ready_to);
                continue;
            }
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
            const bool masked = pos_lo - key0 < CK_BN - 1 || key0 < first_key(a.window, pos_hi);
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
            // p = 2^(s - m_ref) as bf16 pairs over the first 64 columns of S.  All of them by the special-function unit: a quarter by polynomials
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
                if (Z::HALVES && c == 32) {  // (the stores of the first half are done by now)
                    tmem_st_wait();
                    weights_are_there(&p_half[t], half_to);
                }
                tmem_st16(s_addr + c, w);
            }
            float la, lb;
            unpack2(fadd2(fadd2(ls2[0], ls2[1]), fadd2(ls2[2], ls2[3])), la, lb);
            const float sum = la + lb;
            l = sum > CK_JUMP ? CK_AGAIN : l + sum;
            raise = sum > CK_RAISE && sum <= CK_JUMP ? (int)(__float_as_uint(sum) >> 23) - 127 : 0;
            tmem_st_wait();
            weights_are_there(&p_ready[t], ready_to);
        }
        if (ok && n_max > j_lo) ok = ck_wait_warp<PAIR>(&o_done, 0, &abort_flag, a.c.err, TC_TIMEOUT_ACC);
        tc_fence_after();
        const bool any = ok && mine && je[t] > jb[t];  // (the whole query tile)
        // What follows is executed once per CTA, mostly for the first time on its multiprocessor: rolled loops, because every line of code is fetched (unrolled, with the
        // factors of up to seven senders in registers, the end of a CTA took 4.2 us instead of 1.6).
        const int sw = warp - CK_SOFTMAX;
        // The meeting of a pair's CTAs, in place of tiles and rings: the rows of the eight softmax warps belong to the CTAs in equal shares; [sender][row of this CTA][D] sums and,
        // behind them, [sender][row] references and sums of the weights.
        const int own_rows = 2 * CK_BM / share;
        uint8_t* recv = tiles;
        uint8_t* recv_ml = tiles + (share - 1) * own_rows * (D * 4);
        uint8_t* staged = (share > 1 ? recv_ml + (share - 1) * own_rows * 8 : tiles) + sw * (32 * D * 2);  // this warp's 32 rows pass through here
        // What the last key tile asks for: rows meet under references that their sums of weights are near to, so that a factor below 2^-126 is one of nothing.
        const float fold = ex2_approx((float)-raise);
        if (l != CK_AGAIN) l *= fold;
        m_ref += (float)raise;
        float own = fold, L = l, M = m_ref;  // factor of the sums in TMEM, sum of the weights, reference of the row
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
                const int at = (part < owner ? part : part - 1) * own_rows + r_own, peer = rank + (PAIR ? 2 : 1) * (owner - part);
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
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fold);
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
            have = owner == part && mine;
            if (have) {
                senders = share - 1;
                if (!any) M = CK_NONE;
#pragma unroll 1
                for (int p = 0; p < senders; ++p) M = fmaxf(M, reinterpret_cast<const float2*>(recv_ml)[p * own_rows + r_own + lane].x);
                const float w_own = ex2_approx(m_ref - M);
                own = any ? w_own * fold : 0.0f;
                L = !any ? 0.0f : l == CK_AGAIN ? l : l * w_own;
#pragma unroll 1
                for (int p = 0; p < senders; ++p) {
                    const float2 w = sent_factor(p);
                    if (w.y == CK_AGAIN) L = w.y;
                    else if (w.x != 0.0f || w.y != 0.0f) L = fmaf(w.x, w.y, L);
                }
            }
        }
        if (have) {
            const float inv = 1.0f / L;
            bool bad = L == CK_AGAIN;
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
            // (a sum of weights that is a NaN comes from a score that is no number, of a key that the row sees: nothing else would come out of it a second time)
            bad = bad && L == L;
            // rows leave whole, 16 bytes per lane; lane r knows where row r goes (a row that is worked out again does not: the outputs may lie where its query is)
            constexpr int PIECES = D / 8, STEP = 32 / PIECES;
            const int piece = lane % PIECES, in = (int)(row * f.inv_G >> 16);
            const long long goes = query && !bad ? (row0 + token) * a.out_rs + (long long)(hk * a.G + row - in * a.G) * D : -1;
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
            // bf16 pieces) and, where a row is a whole line, in bit 2 (the places of the raw pieces).  The loop over the raw pages stays rolled: unrolled, 335 instead of 231 us for
            // 1000 of 9000 positions at that time (counters: two warps on average were waiting for instructions whenever one was issued).
            const int c4 = lane & 3, second = (lane >> 2) & 1;
            const uint32_t k_u32 = smem_u32(k_smem), v_u32 = smem_u32(v_smem), raw_sc = smem_u32(raw_scales), raw_u32 = smem_u32(raw_smem);
            struct Turn { int row; uint32_t src, dst; };
            // rows of 128 numbers in two slabs (four turns a page), of 64 (two): lines of their own (half of the columns of 128), or two to a line (heads of 64)
            auto wide = [&](int n) {
                const int slab = (lane >> 3) & 1, pair = (n & 1) * 2 + (lane >> 4), r = cw * 16 + (n >> 1) * 8 + (second ? pair ^ 5 : pair);
                return Turn{r, (uint32_t)(r * 128 + (((slab * 4 + c4) ^ (r & 7)) << 4)), slab * Z::K_SLAB + r * 128 + (((c4 * 2) ^ (r & 7)) << 4)};
            };
            auto narrow = [&](int n) {
                const int r = cw * 16 + n * 8 + (lane >> 3) * 2 + second, line = r >> 1;
                return Turn{r, (uint32_t)(D == 64 ? line * 128 + ((((r & 1) * 4 + c4) ^ (line & 7)) << 4) : r * 64 + ((c4 ^ (line & 3)) << 4)), (uint32_t)(r * 128 + (((c4 * 2) ^ (r & 7)) << 4))};
            };
            // numbers of rows from .. until - 1 of a page, zeros elsewhere
            auto convert = [&](auto at, auto turns, uint32_t raw, uint32_t scales, uint32_t to, int from, int until) {
                constexpr int N = decltype(turns)::value;
                uint4 w[N];
                uint32_t scale[N];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const Turn x = at(n);
                    w[n] = lds128(raw + x.src);
                    scale[n] = lds16(scales + x.row * 2);
                }
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const Turn x = at(n);
                    const uint32_t sc = x.row < from || x.row >= until ? 0u : scale[n] * 0x00010001u;
                    sts128(to + x.dst, make_uint4(q8_value2(__byte_perm(w[n].x, 0, 0x1100), sc), q8_value2(__byte_perm(w[n].x, 0, 0x3322), sc),
                                                  q8_value2(__byte_perm(w[n].y, 0, 0x1100), sc), q8_value2(__byte_perm(w[n].y, 0, 0x3322), sc)));
                    sts128(to + (x.dst ^ 16), make_uint4(q8_value2(__byte_perm(w[n].z, 0, 0x1100), sc), q8_value2(__byte_perm(w[n].z, 0, 0x3322), sc),
                                                         q8_value2(__byte_perm(w[n].w, 0, 0x1100), sc), q8_value2(__byte_perm(w[n].w, 0, 0x3322), sc)));
                }
            };
            constexpr std::integral_constant<int, 4> four{};
            constexpr std::integral_constant<int, 2> two{};
            bool ok = true;
            for (int j = j_lo; j < n_max && ok; ++j) {
                const int i = j - j_lo, s = i % ST;
#pragma unroll 1
                for (int slot = 0; slot < Z::SLOTS; ++slot) {
                    const int value = PAIR ? slot > 0 : slot >> 1, half = PAIR ? (slot ? slot - 1 : 0) : slot & 1;
                    const bool first = half == 0, last = half == 1 || (PAIR && !value);
                    if (first && i >= ST && !ck_wait_warp<PAIR>(value ? &v_empty[s] : &k_empty[s], ((i / ST) & 1) ^ 1, &abort_flag, a.c.err, TC_TIMEOUT_EMPTY)) { ok = false; break; }
                    if (!mbar_wait_warp(&raw_full[slot], i & 1, &abort_flag, a.c.err, TC_TIMEOUT_FULL)) { ok = false; break; }
                    const uint32_t raw = raw_u32 + Z::raw_at(slot), scales = raw_sc + slot * (JSM_PAGE_SIZE * 2);
                    const uint32_t to = (value ? v_u32 : k_u32) + s * Z::KV + half * (JSM_PAGE_SIZE * 128);
                    // values that no row sees become zeros: a weight of zero meets a number
                    const int key0 = base + j * CK_BN + half * JSM_PAGE_SIZE, from = value ? lo - key0 : -1, until = value ? end - key0 : JSM_PAGE_SIZE;
                    if constexpr (D == 64) convert(narrow, two, raw, scales, to, from, until);
                    else if constexpr (!PAIR) convert(wide, four, raw, scales, to, from, until);
                    else if (value) convert(narrow, two, raw, scales, to, from, until);
                    else convert(wide, four, raw, scales, to, from, until);
                    if (last) fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&raw_empty[slot]);
                        if (last) mbar_arrive(value ? &v_full[s] : &k_full[s]);
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
    if (PAIR) {
        ck_cluster_arrive();
        ck_cluster_wait();  // the leader's products and arrivals have reached the other CTA, and the other's the leader
    }
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
        else tmem_dealloc(tmem_base, 512);
    }
}

// clusters of S CTAs that the chip holds at once (15 of eight, 33 of four, although it has 148 multiprocessors)
template <int D, bool Q8, bool PAIR>
static int flash_capacity(int S) {
    static std::mutex mu;
    static int known[64][9];  // per device and instantiation
    int dev = -1;
    const int guess = S == 1 ? sm_count() : sm_count() / S * 3 / 4;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return guess;
    std::lock_guard<std::mutex> lock(mu);
    if (known[dev][S] == 0) {
        static DeviceOnce once;
        const cudaError_t allowed = allow_shared(once, chunk_flash_kernel<D, Q8, PAIR>, (int)FlashSizes<D, Q8, PAIR>::SMEM);
        if (allowed != cudaSuccess) return guess;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(S * 256);
        cfg.blockDim = dim3(FlashSizes<D, Q8, PAIR>::THREADS);
        cfg.dynamicSmemBytes = FlashSizes<D, Q8, PAIR>::SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = S;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, chunk_flash_kernel<D, Q8, PAIR>, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = guess;
        }
        known[dev][S] = n;
    }
    return known[dev][S];
}

// How a call is shared out, and what it may take (us).
struct FlashPlan {
    long long units;  // at most
    int cluster, walk_tiles;
    float cost;
};
template <int D, bool Q8, bool PAIR>
static FlashPlan flash_plan(const ChunkArgs& a) {
    constexpr int CTAS = PAIR ? 2 : 1;  // of a unit
    const long long tokens = 2ll * CTAS * (CK_BM / a.G), per_seq = (a.max_new + tokens - 1) / tokens;
    FlashPlan p{std::min(per_seq * a.c.n_seqs, a.T / tokens + a.c.n_seqs) * a.c.Hkv, 1, INT_MAX, 0.0f};
    // Units that share the key tiles of theirs.  A key tile takes about 2 us (of an 8-bit cache 2.4, a pair 2.1), what is around the walk 6 us (a pair 7), a meeting 3 us: the longest
    // unit, or the chip's share of all and half a unit's time for the uneven end.  On average the query tiles of one sequence see what lies before the middle of its new tokens, those of many
    // sequences perhaps half of that.
    constexpr float TILE = PAIR ? 2.1f : Q8 ? 2.4f : 2.0f, AROUND = PAIR ? 7.0f : 6.0f;
    long long keys = a.max_context, mean = a.max_context - a.max_new / 2;
    if (a.c.n_seqs > 1) mean /= 2;
    if (a.window > 0) { keys = std::min(keys, (long long)a.window + tokens); mean = std::min(mean, keys); }
    const int key_tiles = (int)((keys + CK_BN - 1) / CK_BN);
    const float mean_tiles = (float)mean / CK_BN, likely = a.c.n_seqs > 1 ? (float)(a.T / tokens + a.c.n_seqs / 2 + 1) * a.c.Hkv : (float)p.units;
    for (int S = 1; S * CTAS <= 8; S *= 2) {
        if (S > 1 && key_tiles < 2 * S) break;
        const int cap = flash_capacity<D, Q8, PAIR>(S * CTAS) * S, walk = (key_tiles + S - 1) / S;
        const float around = AROUND + (S > 1 ? 3.0f : 0.0f), longest = around + TILE * walk;
        const float units = likely * std::max(1.0f, mean_tiles / walk), one = around + TILE * std::min(mean_tiles, (float)walk);
        const float cost = units <= cap ? longest : std::max(longest, one * (units / cap + 0.5f));
        // (a sharing that promises less than a tenth is not taken: 16 sequences of one token to 1000, 67 promised for 70, took 75 us instead of 69)
        if (S == 1 || cost < 0.9f * p.cost) { p.cost = cost; p.cluster = S; p.walk_tiles = walk; }
    }
    return p;
}

template <int D, bool Q8, bool PAIR>
static jsm_status flash_launch(const ChunkArgs& a, const FlashPlan& p, int few_tokens, cudaStream_t st) {
    using Z = FlashSizes<D, Q8, PAIR>;
    constexpr int CTAS = PAIR ? 2 : 1;
    const FlashArgs f{a, few_tokens, CK_BM / a.G, 2 * CTAS, p.cluster, p.walk_tiles, (65536u + a.G - 1) / a.G};
    if (p.units * f.cluster * CTAS > INT32_MAX) JSM_FAIL(JSM_UNSUPPORTED, "jsm_attn_chunk: %lld tiles of queries", p.units);
    static DeviceOnce once;
    const cudaError_t allowed = allow_shared(once, chunk_flash_kernel<D, Q8, PAIR>, (int)Z::SMEM);
    JSM_CUDA_CHECK(allowed);
    CUtensorMap mq, mkv, mhalf;
    jsm_status s = make_tmap_bf16_3d(&mq, a.q, D, a.Hq, a.T, D, a.q_rs, 64, a.G, f.tile_tokens);
    if (s != JSM_OK) return s;
    const uint64_t rows = (uint64_t)a.c.n_pages * 2 * a.c.Hkv * JSM_PAGE_SIZE;
    s = Q8 ? make_tmap_u8_lines(&mkv, a.c.pool, rows * D / 128, JSM_PAGE_SIZE * D / 128) : make_tmap_bf16_2d(&mkv, a.c.pool, rows, D, D, JSM_PAGE_SIZE, 64);
    if (s != JSM_OK) return s;
    mhalf = mkv;
    if (Q8 && PAIR) s = make_tmap_u8_halves(&mhalf, a.c.pool, rows, JSM_PAGE_SIZE);
    if (s != JSM_OK) return s;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.units * f.cluster * CTAS));
    cfg.blockDim = dim3(Z::THREADS);
    cfg.dynamicSmemBytes = Z::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = f.cluster * CTAS;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = chained_launch_enabled() ? attr : attr + 1;
    cfg.numAttrs = (chained_launch_enabled() ? 1 : 0) + (f.cluster * CTAS > 1 ? 1 : 0);
    const cudaError_t launched = cudaLaunchKernelEx(&cfg, chunk_flash_kernel<D, Q8, PAIR>, mq, mkv, mhalf, f);
    JSM_CUDA_CHECK(launched);
    JSM_LAUNCH_CHECK();
    return JSM_OK;
}

template <int D, bool Q8>
static jsm_status flash_launch(const ChunkArgs& a, int few_tokens, cudaStream_t st) {
    const FlashPlan one = flash_plan<D, Q8, false>(a);
    if constexpr (Q8 && D == 128) {
        const FlashPlan two = flash_plan<D, Q8, true>(a);
        if (two.cost < one.cost) return flash_launch<D, Q8, true>(a, two, few_tokens, st);
    }
    return flash_launch<D, Q8, false>(a, one, few_tokens, st);
}

jsm_status chunk_flash_launch(const ChunkArgs& a, int few_tokens, cudaStream_t st) {
    if (a.c.D == 64) return a.c.scales ? flash_launch<64, true>(a, few_tokens, st) : flash_launch<64, false>(a, few_tokens, st);
    return a.c.scales ? flash_launch<128, true>(a, few_tokens, st) : flash_launch<128, false>(a, few_tokens, st);
}

}  // namespace jsm
