// Product of the 8-bit linear path: out[s][n] (+)= (sum_k q_w[n][k] q_x[s][k]) * scale_w[n] * scale_x[s], int8 operands
// with one scale per weight row and one per token, the sum exact in int32.
//
// The weight rows are the MMA's M (128 TMEM lanes), the tokens its N (TMEM columns): tcgen05.mma kind::i8, 128 x NTOK x 32.
// With the channel on the lane a warp's store of one token is 128 contiguous bytes, and a short batch costs no more
// than its own columns.  Both planes are stored as swizzled shared-memory tiles (common.cuh), so an operand is one
// contiguous copy: 16 KiB of weights and NTOK * 128 bytes of activations per 128-column block.
//
// Few tokens: the time is the weights' way from HBM, and what counts is how many bytes are in flight on how many SMs.
// A tile of 128 rows is cut along K over the CTAs of a cluster; integer partial sums meet through distributed shared
// memory (no workspace, no atomics, any order gives the same bits), every CTA finishing its share of the tokens.
// The weight copies of the first stages are issued before the wait on the previous kernel of the stream (programmatic
// dependent launch): weights are written once, at upload, which synchronises.
//
// Many tokens: bound by the tensor cores, so a pair of CTAs works on one tile of 256 rows x NT tokens (cta_group::2: each
// SM holds half of either operand, which halves the shared-memory traffic per product), persistent over the tiles, two
// accumulators in TMEM so that one tile is scaled and stored while the next is summed.  Its copies go through tensor maps (made
// with the handles): of a copy's forms only that one may count its bytes at a barrier of the other CTA of the pair.
//
// Measured (back to back in a graph, us; weight bytes per second or operations per second):
//   1 x 2048 x 151669   47.0 (6.6 TB/s, the copy bandwidth)      4 x 5120 x 34816    27.5 (6.5 TB/s)
//   1 x 4096 x 4096      4.3 (weights in L2)                     16 x 4096 x 24576   17.7 (5.7 TB/s)
//   32 x 17408 x 5120   16.4 (5.4 TB/s)                          77 x 12288 x 4096   14.5 (3.5 TB/s)
//   512 x 4096 x 24576  44.2 (2 330 TOP/s)                       4096 x 5120 x 17408  236 (3 090 TOP/s)
// The last two before the GPU throttles.  After two seconds of the last it takes 273 (2 680 TOP/s) at the 1000 W limit and a sampled
// median of 1.37 GHz: 373 000 cycles, of which its MMAs are 307 000 (15 rounds of tiles x 20 stages x 1 024).
// Between 33 and 128 tokens a third of the time is not streaming: from a kernel's end to its successor's wait 2 us, the
// exchange of the partial sums 2 us (a CTA stores about 8 bytes a clock into its neighbours), barrier and output 2 us.
//
// Every wait on an mbarrier is bounded; on expiry the CTA records a status code, drains its copies, frees its TMEM and
// returns (its cluster neighbours still meet it at the cluster barriers).
#include <algorithm>

#include "tc_common.cuh"

namespace hb200 {

namespace {

constexpr int W_TILE = 16384;  // 128 rows x 128 bytes
constexpr int MAX_SPLIT = 8;   // portable cluster size

// Only once this CTA has its TMEM: a dependent kernel's CTA that came first to the SM's columns would wait for this grid's end, and
// this one for the columns.
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Untiled bulk copy: addresses and size are multiples of 16 bytes by the planes' layout.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
                 "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
// True in one lane of a converged warp.  The roles below run their loops with the whole warp and elect a lane only around
// the issuing instructions: inside a branch on the lane number those (their operands are warp-uniform registers) and
// the barrier tests cost several times as much.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "elect.sync _|P, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t}"
        : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_smem(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void peer_st4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// mbar_wait by a converged warp, whose lanes leave it together and agree on the answer.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
    for (uint32_t i = 0; i < SPIN_LIMIT; i++) {
        if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
        if ((i & 7) == 7 && __any_sync(0xffffffffu, *abort_flag)) return false;
    }
    *abort_flag = 1;
    atomicCAS(status, 0, code);
    return false;
}

// The same with acquire at cluster scope, for barriers that the other CTA of a pair (or its copies) arrives at.
__device__ __forceinline__ bool mbar_try_cluster(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_pair(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
    for (uint32_t i = 0; i < SPIN_LIMIT; i++) {
        if (__all_sync(0xffffffffu, mbar_try_cluster(bar, parity))) return true;
        if ((i & 7) == 7 && __any_sync(0xffffffffu, *abort_flag)) return false;
    }
    *abort_flag = 1;
    atomicCAS(status, 0, code);
    return false;
}

// The last commit of a CTA, awaited with a limit whether or not the CTA is giving up.
__device__ __forceinline__ void await_mmas(uint32_t bar) {
    for (uint32_t i = 0; i < SPIN_LIMIT && !__all_sync(0xffffffffu, mbar_try(bar, 0)); i++) {}
}

// The order of the two multiplications keeps an intermediate of tiny scales out of the subnormals.
__device__ __forceinline__ float scaled(int acc, float sw, float sx) { return __fmul_rn(__fmul_rn(__int2float_rn(acc), sw), sx); }

template <int NTOK>
constexpr uint32_t idesc_i8() {  // D = S32, A and B signed int8, both K-major, M = 128, N = NTOK
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NTOK >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// A CTA's share of the tokens of a tile that `split` CTAs finish together, in fours.
__host__ __device__ constexpr int token_share(int n_tok, int split) { return ((n_tok + split - 1) / split + 3) / 4 * 4; }
constexpr int part_bytes(int ntok) {
    int most = 0;
    for (int s = 2; s <= MAX_SPLIT; s++) {
        const int b = s * 128 * token_share(ntok, s) * 4;
        if (b > most) most = b;
    }
    return most;
}

template <int NTOK>
struct SplitCfg {
    static constexpr int X_TILE = NTOK * 128;
    static constexpr int STAGE = W_TILE + X_TILE;
    // two CTAs per SM
    static constexpr int STAGES = NTOK <= 16 ? 5 : 4;
    // Partial sums of the cluster's CTAs: memory of their own at few tokens, else the ring's once it has run dry.
    static constexpr bool OWN_PART = NTOK <= 32;
    static constexpr int PART = part_bytes(NTOK);
    static constexpr int SMEM = STAGES * STAGE + (OWN_PART ? PART : 0) + 1024;
    static constexpr uint32_t COLS = NTOK < 32 ? 32 : NTOK;
    static_assert(OWN_PART || PART <= STAGES * STAGE, "partial sums fit the ring");
};

// grid (split, token tiles, row tiles), cluster (split, 1, 1): rank r of a cluster takes blocks [kb * r / split, kb * (r + 1) / split).
template <int NTOK>
__global__ void __launch_bounds__(128) i8_split_kernel(const I8Product p) {
    using C = SplitCfg<NTOK>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ unsigned char dyn[];
    __shared__ uint64_t full[STAGES], empty[STAGES], done;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, failed, s_failed[MAX_SPLIT];
    __shared__ float s_sx[NTOK];
    __shared__ alignas(16) float s_sw[128];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = gridDim.x, rank = blockIdx.x;
    const int tok0 = blockIdx.y * NTOK, row_tile = blockIdx.z, row0 = row_tile * 128;
    const int n_tok = min(NTOK, p.n_tok - tok0);
    const int k0 = (int)((long long)p.kb * rank / split), k1 = (int)((long long)p.kb * (rank + 1) / split), nk = k1 - k0;
    const uint32_t ring = (smem_u32(dyn) + 1023u) & ~1023u;
    const uint32_t x_bytes = (uint32_t)((n_tok + 7) / 8) * 1024;  // whole groups of eight tokens; other columns of the tile are not stored
    const int8_t* wp = p.w + ((size_t)row_tile * p.kb + k0) * W_TILE;
    const int8_t* xp = p.a + (size_t)k0 * p.a_kb_stride + (size_t)tok0 * 128;

    if (tid == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        mbar_init(smem_u32(&done), 1);
        abort_flag = failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = 0; i < nk && i < STAGES; i++) {
            mbar_expect_tx(smem_u32(&full[i]), W_TILE + x_bytes);
            bulk_load(ring + i * C::STAGE, wp + (size_t)i * W_TILE, W_TILE, smem_u32(&full[i]));
        }
    }
    __syncwarp();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(C::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // This CTA runs: its memory may be written (awaited far below).  Relaxed: a release would wait for the bulk copies.
    if (C::OWN_PART && split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_trigger();
    pdl_wait();

    if (warp == 0) {
        if (elect_one())
            for (int i = 0; i < nk && i < STAGES; i++)
                bulk_load(ring + i * C::STAGE + W_TILE, xp + (size_t)i * p.a_kb_stride, x_bytes, smem_u32(&full[i]));
        __syncwarp();
        int issued = min(nk, STAGES);
        for (int i = STAGES; i < nk; i++) {
            const int s = i % STAGES;
            if (!mbar_wait_warp(smem_u32(&empty[s]), (uint32_t)(i / STAGES - 1) & 1u, &abort_flag, p.status, 60)) break;
            const uint32_t dst = ring + s * C::STAGE;
            if (elect_one()) {
                mbar_expect_tx(smem_u32(&full[s]), W_TILE + x_bytes);
                bulk_load(dst, wp + (size_t)i * W_TILE, W_TILE, smem_u32(&full[s]));
                bulk_load(dst + W_TILE, xp + (size_t)i * p.a_kb_stride, x_bytes, smem_u32(&full[s]));
            }
            __syncwarp();
            issued = i + 1;
        }
        if (*(volatile int*)&abort_flag) {  // nothing may still be on its way into this CTA's memory when it ends
            for (int i = max(0, issued - STAGES); i < issued; i++)
                for (uint32_t t = 0; t < SPIN_LIMIT && !mbar_try(smem_u32(&full[i % STAGES]), (uint32_t)(i / STAGES) & 1u); t++) {}
        }
        __syncwarp();
    } else if (warp == 1) {
        for (int i = 0; i < nk; i++) {
            const int s = i % STAGES;
            if (!mbar_wait_warp(smem_u32(&full[s]), (uint32_t)(i / STAGES) & 1u, &abort_flag, p.status, 61)) break;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t ad = make_desc(ring + s * C::STAGE), bd = make_desc(ring + s * C::STAGE + W_TILE);
#pragma unroll
                for (int j = 0; j < 4; j++) mma_i8(tmem, ad + 2 * j, bd + 2 * j, idesc_i8<NTOK>(), (i | j) != 0);
                tc_commit(smem_u32(&empty[s]));
            }
            __syncwarp();
        }
        // also after a wait that ran out: no MMA may still read this CTA's memory when it ends
        if (elect_one()) tc_commit(smem_u32(&done));
        __syncwarp();
        await_mmas(smem_u32(&done));
        if (*(volatile int*)&abort_flag || !mbar_try(smem_u32(&done), 0)) {
            atomicCAS(p.status, 0, 62);
            failed = 1;
        }
#ifdef HB200_BOUNDS
        if (p.report_rank == rank + 1) {  // the self-test: this CTA says so although nothing ran out
            atomicCAS(p.status, 0, 62);
            failed = 1;
        }
#endif
        __syncwarp();
    } else if (warp == 2) {
        for (int t = lane; t < NTOK; t += 32) s_sx[t] = t < n_tok ? p.sx[tok0 + t] : 0.f;
    } else {
        for (int r = lane; r < 128; r += 32) s_sw[r] = row0 + r < p.n_rows ? p.sw[row0 + r] : 0.f;
    }
    __syncthreads();
    tc_fence_after();
    bool ok = !failed;

    const int row = row0 + warp * 32 + lane;
    const uint32_t tm = tmem + ((uint32_t)(warp * 32) << 16);
    if (split == 1) {
        const float sw = s_sw[warp * 32 + lane];
        float* out = p.out + (size_t)tok0 * p.ld_out + row;
        for (int c0 = 0; c0 < n_tok; c0 += 16) {
            uint32_t v[16];
            tmem_ld16(tm + c0, v);
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (ok && row < p.n_rows && c0 + j < n_tok) {
                    float* o = out + (size_t)(c0 + j) * p.ld_out;
                    const float r = scaled((int)v[j], sw, s_sx[c0 + j]);
                    *o = p.accumulate ? __fadd_rn(*o, r) : r;
                }
            __syncwarp();  // the lanes of rows past the end rejoin before the next TMEM load
        }
    } else {
        // Every CTA finishes its share of the tokens: all store their sums of them into its memory, [sender][four tokens]
        // [row], 512 neighbouring bytes a warp (stores do not wait for an answer: loads from the others took 6 000 cycles at
        // 77 tokens; single tokens a store 2 400; rows of all tokens, 16 bytes here and there, more than that).
        const int share = token_share(n_tok, split);
        const uint32_t part = C::OWN_PART ? ring + STAGES * C::STAGE : ring;
        const uint32_t mine = part + (uint32_t)(rank * share * 512 + tid * 16);
        if (!C::OWN_PART) cluster_arrive();  // this CTA's copies have landed and been read
        cluster_wait();                      // the others' memory is there (and free)
        if (tid < split)  // a CTA that gave up has no sums: nobody stores any of this tile then
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_smem(smem_u32(&s_failed[rank]), tid)), "r"(failed) : "memory");
        __syncwarp();
        int owner = 0, at = 0;
        for (int c0 = 0; c0 < n_tok; c0 += 16) {
            uint32_t v[16];
            tmem_ld16(tm + c0, v);
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                if (c0 + j < n_tok) peer_st4(peer_smem(mine, owner) + at * 512, v[j], v[j + 1], v[j + 2], v[j + 3]);
                at += 4;
                if (at == share) { at = 0; owner = min(owner + 1, split - 1); }
            }
        }
        cluster_sync();
        ok = !__any_sync(0xffffffffu, lane < split && s_failed[lane & (MAX_SPLIT - 1)]);
        const int first = rank * share, n_mine = min(share, n_tok - first);
        const int4* sums = reinterpret_cast<const int4*>(dyn + (part - smem_u32(dyn))) + tid;
        const float sw = s_sw[tid];
        float* o = p.out + (size_t)(tok0 + first) * p.ld_out + row;
        for (int t = 0; t < n_mine; t += 4) {
            int4 s = make_int4(0, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < MAX_SPLIT; r++)
                if (r < split) {
                    const int4 q = sums[(r * share + t) * 32];
                    s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w;
                }
            const int q[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (ok && row < p.n_rows && t + j < n_mine) {
                    const float f = scaled(q[j], sw, s_sx[first + t + j]);
                    float* d = o + (size_t)(t + j) * p.ld_out;
                    *d = p.accumulate ? __fadd_rn(*d, f) : f;
                }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
    }
}

// ---- a pair of CTAs per tile: many tokens ---------------------------------------------------------------------------

template <int NT>
struct PairCfg {
    static constexpr int X_TILE = NT / 2 * 128;  // this CTA's half of the tokens
    // Two 128-column blocks a stage (the last stage of a tile may hold one): a barrier test costs the issuing warp some
    // 160 cycles even when it succeeds; with one block a stage (256 cycles of MMAs at 128 tokens) the tensor pipe waited
    // for the issue.
    static constexpr int STAGE = 2 * (W_TILE + X_TILE);
    static constexpr int STAGES = NT == 256 ? 3 : 4;
    static constexpr int SMEM = STAGES * STAGE + 1024;
    static constexpr uint32_t COLS = 2 * NT;  // two accumulators
};
constexpr int PAIR_EPI_WARPS = 8;  // two per TMEM lane quarter, each half of the tile's tokens
constexpr int PAIR_THREADS = 32 * (2 + PAIR_EPI_WARPS);  // producer, MMA issue (or relay), epilogue
// Token tiles that are walked together: their activations stay in L2 while the weights go by (16 x 256 tokens of
// 17408 columns are 71 MB), and the weights are read once per group.
constexpr int TOK_GROUP = 16;

// A block of 128 columns of a plane, rows `row` .. of the map's box, into this CTA's memory; its bytes count at `bar`, a barrier of
// either CTA of the pair.  What a copy wrote is visible to whoever acquires the completed phase at cluster scope, so the
// leader's one barrier per stage covers both CTAs' halves of it.
__device__ __forceinline__ void pair_load(uint32_t dst, const CUtensorMap* map, int row, int block, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(0), "r"(row), "r"(block), "r"(bar)
        : "memory");
}
// Arrival at a barrier of the other CTA, released at cluster scope.
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives at the barrier of this offset in both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
          "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]),
          "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}

// 32 tokens of a row: a warp's store is 32 neighbouring rows of one token.  The output of a long prompt is larger than L2
// and not read back here: stored for early eviction.
template <bool ACC, bool PART>
__device__ __forceinline__ void store_cols(float* o, size_t ld, const uint32_t (&v)[32], float sw, float sx, bool live, int cols) {
    float r[32];
#pragma unroll
    for (int j = 0; j < 32; j++) r[j] = scaled((int)v[j], sw, __shfl_sync(0xffffffffu, sx, j));
    if (!live) return;
    if (ACC) {
#pragma unroll
        for (int j = 0; j < 32; j++)
            if (!PART || j < cols) r[j] = __fadd_rn(__ldcs(o + (size_t)j * ld), r[j]);
    }
#pragma unroll
    for (int j = 0; j < 32; j++) {
        if (PART && j >= cols) break;
        __stcs(o, r[j]);
        o += ld;
    }
}

struct PairTile {
    int row_tile, tok0;  // this CTA's 128-row tile, first token of the pair's tile
};
// Tiles in groups of TOK_GROUP token tiles, the token tile fastest inside a group.
template <int NT>
__device__ __forceinline__ PairTile pair_tile(int t, int row_pairs, int tok_tiles, int rank) {
    const int group = t / (TOK_GROUP * row_pairs), first = group * TOK_GROUP;
    const int width = min(TOK_GROUP, tok_tiles - first), i = t - first * row_pairs;
    PairTile r;
    r.tok0 = (first + i % width) * NT;
    r.row_tile = (i / width) * 2 + rank;
    return r;
}

template <int NT, bool ACC>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
    i8_pair_kernel(const I8Product p, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, int row_pairs, int tok_tiles) {
    using C = PairCfg<NT>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ unsigned char dyn[];
    // full (leader): both CTAs' copies of a stage; empty: the stage may be refilled; acc_full / acc_empty: an accumulator is
    // complete / has been read (leader: by both CTAs' epilogue warps); drained: no MMA is under way any more
    __shared__ uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, n_tiles = row_pairs * tok_tiles;
    const int last_row_tile = (p.n_rows + 127) / 128 - 1;
    const uint32_t ring = (smem_u32(dyn) + 1023u) & ~1023u;
    const uint32_t full0 = smem_u32(&full[0]), empty0 = smem_u32(&empty[0]);

    // Rank r's half of a tile's tokens: none of them may be there, else a whole box is read (rows behind the plane's are zeros).
    const auto half_live = [&](int tok0, int r) { return tok0 + r * (NT / 2) < p.n_tok; };
    const auto stage_bytes = [&](int tok0, int blocks) {  // of both CTAs
        return (uint32_t)blocks * (2 * W_TILE + (half_live(tok0, 1) ? 2 : 1) * C::X_TILE);
    };
    const auto w_block = [&](const PairTile& t) { return min(t.row_tile, last_row_tile) * p.kb; };

    const PairTile t0 = pair_tile<NT>(pair, row_pairs, tok_tiles, rank);
    const int steps = (p.kb + 1) / 2;     // stages of a tile
    const int ahead = min(steps, STAGES);  // stages whose weights are fetched before the wait on the previous kernel
    if (tid == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(smem_u32(&acc_full[a]), 1);
            mbar_init(smem_u32(&acc_empty[a]), 2 * PAIR_EPI_WARPS);
        }
        mbar_init(smem_u32(&drained), 1);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(C::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync();  // both CTAs' barriers exist before either signals the other
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const uint32_t leader_full0 = peer_smem(full0, 0);
    if (warp == 0 && elect_one()) {
        for (int k = 0; k < ahead; k++) {
            const int blocks = min(2, p.kb - 2 * k);
            if (rank == 0) mbar_expect_tx(full0 + k * 8, stage_bytes(t0.tok0, blocks));
            for (int b = 0; b < blocks; b++)
                pair_load(ring + k * C::STAGE + b * W_TILE, &w_map, 0, w_block(t0) + 2 * k + b, leader_full0 + k * 8);
        }
    }
    __syncwarp();
    pdl_trigger();
    pdl_wait();

    if (warp == 0) {
        int it = 0, s = 0;
        uint32_t phase = 1;  // parity of the `empty` completion before the one this use makes
        bool ok = true;
        for (int t = pair; t < n_tiles && ok; t += pairs) {
            const PairTile tl = pair_tile<NT>(t, row_pairs, tok_tiles, rank);
            const bool live = half_live(tl.tok0, rank);
            const int w0 = w_block(tl), x_row = tl.tok0 + (int)rank * (NT / 2);
            for (int k = 0; k < p.kb; k += 2, it++) {
                if (it >= STAGES) ok = mbar_wait_pair(empty0 + s * 8, phase, &abort_flag, p.status, 63);
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t dst = ring + s * C::STAGE, bar = leader_full0 + s * 8;
                    const int blocks = min(2, p.kb - k);
                    if (it >= ahead) {
                        if (rank == 0) mbar_expect_tx(full0 + s * 8, stage_bytes(tl.tok0, blocks));
                        pair_load(dst, &w_map, 0, w0 + k, bar);
                        if (blocks == 2) pair_load(dst + W_TILE, &w_map, 0, w0 + k + 1, bar);
                    }
                    if (live) {
                        pair_load(dst + 2 * W_TILE, &x_map, x_row, k, bar);
                        if (blocks == 2) pair_load(dst + 2 * W_TILE + C::X_TILE, &x_map, x_row, k + 1, bar);
                    }
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; phase ^= 1; }
            }
        }
        // Nothing may still be on its way into either CTA's memory when they end: both stay until the leader has seen the copies land
        // (a stage that the other CTA never filled runs into the limit).
        if (rank == 0 && *(volatile int*)&abort_flag) {
            for (int i = max(0, it - STAGES); i < it; i++)
                for (uint32_t n = 0; n < SPIN_LIMIT && !mbar_try_cluster(full0 + i % STAGES * 8, (uint32_t)(i / STAGES) & 1u); n++) {}
        }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {
        // D = S32, A and B signed int8, both K-major, M = 256 over the pair, N = NT
        constexpr uint32_t IDESC = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
        const uint64_t ad0 = make_desc(ring), bd0 = make_desc(ring + 2 * W_TILE);
        int n = 0, s = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = pair; t < n_tiles && ok; t += pairs, n++) {
            const int a = n & 1;
            if (n >= 2) {
                ok = mbar_wait_pair(smem_u32(&acc_empty[a]), (uint32_t)(n / 2 - 1) & 1u, &abort_flag, p.status, 64);
                if (!ok) break;
                tc_fence_after();
            }
            for (int k = 0; k < p.kb; k += 2) {
                ok = mbar_wait_pair(full0 + s * 8, phase, &abort_flag, p.status, 65);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t ad = ad0 + (uint32_t)(s * (C::STAGE >> 4)), bd = bd0 + (uint32_t)(s * (C::STAGE >> 4));
#pragma unroll
                    for (int j = 0; j < 4; j++) mma_i8_pair(tmem + a * NT, ad + 2 * j, bd + 2 * j, IDESC, (k | j) != 0);
                    if (k + 1 < p.kb) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            mma_i8_pair(tmem + a * NT, ad + (W_TILE >> 4) + 2 * j, bd + (C::X_TILE >> 4) + 2 * j, IDESC, 1);
                    }
                    commit_pair(empty0 + s * 8);
                    if (k + 2 >= p.kb) commit_pair(smem_u32(&acc_full[a]));
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; phase ^= 1; }
            }
        }
        // also after a wait that ran out: no MMA may still read either CTA's memory when they end
        if (elect_one()) commit_pair(smem_u32(&drained));
        __syncwarp();
    } else if (warp >= 2) {
        const int q = warp & 3;                      // TMEM lane quarter of this warp
        const int half = (warp - 2) / 4 * (NT / 2);  // its first token of the tile
        const uint32_t leader_empty0 = peer_smem(smem_u32(&acc_empty[0]), 0);
        int n = 0;
        for (int t = pair; t < n_tiles; t += pairs, n++) {
            const int a = n & 1;
            const PairTile tl = pair_tile<NT>(t, row_pairs, tok_tiles, rank);
            const int row = tl.row_tile * 128 + q * 32 + lane;
            const bool live = row < p.n_rows;
            const float sw = live ? p.sw[row] : 0.f;
            if (!mbar_wait_pair(smem_u32(&acc_full[a]), (uint32_t)(n / 2) & 1u, &abort_flag, p.status, 67)) break;
            tc_fence_after();
            const uint32_t tm = tmem + a * NT + half + ((uint32_t)(q * 32) << 16);
            const int n_tok = min(NT / 2, p.n_tok - tl.tok0 - half);
            const float* sxs = p.sx + tl.tok0 + half;
            float* out = p.out + (size_t)(tl.tok0 + half) * p.ld_out + row;
            for (int c0 = 0; c0 < n_tok; c0 += 32) {
                uint32_t v[32];
                const float sx = c0 + lane < n_tok ? sxs[c0 + lane] : 0.f;
                tmem_ld32(tm + c0, v);
                float* o = out + (size_t)c0 * p.ld_out;
                if (c0 + 32 <= n_tok) {
                    store_cols<ACC, false>(o, p.ld_out, v, sw, sx, live, 32);
                } else {
                    store_cols<ACC, true>(o, p.ld_out, v, sw, sx, live, n_tok - c0);
                }
                __syncwarp();  // the lanes of rows past the end rejoin before the next TMEM load
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(leader_empty0 + a * 8);
        }
        __syncwarp();
    }
    __syncthreads();
    if (warp == 1) await_mmas(smem_u32(&drained));
    tc_fence_before();
    cluster_sync();  // the other CTA may still read this one's operands or signal its barriers
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
    }
}

template <int NT>
int launch_pair(const I8Product& p, int sm_count, cudaStream_t st) {
    const int row_pairs = (p.n_rows + 255) / 256, tok_tiles = (p.n_tok + NT - 1) / NT;
    const long long tiles = (long long)row_pairs * tok_tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (unsigned)std::min<long long>(tiles, sm_count / 2));
    cfg.blockDim = dim3(PAIR_THREADS);
    cfg.dynamicSmemBytes = PairCfg<NT>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HB_CUDA(cudaLaunchKernelEx(&cfg, p.accumulate ? i8_pair_kernel<NT, true> : i8_pair_kernel<NT, false>, p, *static_cast<const CUtensorMap*>(p.w_map),
                               *static_cast<const CUtensorMap*>(NT == 256 ? p.x_map_n256 : p.x_map_n128), row_pairs, tok_tiles));
    return 0;
}

struct Plan {
    int ntok, split;  // split 0: the pair kernel
};

int g_sm_count = 148;
// Clusters of the split kernel resident at once, by size: twice what the occupancy query says (it counts one CTA per SM,
// two run).  These are a B200's, replaced by the device's own when the library is initialised.
int g_clusters[MAX_SPLIT + 1] = {0, 296, 148, 90, 66, 52, 44, 30, 30};

// Which kernel, with which tile and how many CTAs along K.
//   split   one token tile of 16, 32 or 64 where that covers the batch.  As many CTAs per tile as keep all clusters
//           resident at once: measured, us, at 1 / 2 / 3 / 4 / 5 / 6 / 8 CTAs along K: 32 tokens of 17408 x 5120 (40 tiles)
//           - / - / 19.3 / 17.8 / 17.2 / 16.5 / 22.3 (at 8 a part of the clusters waits), 16 of 4096 x 24576 (192 tiles)
//           18.0 / 22.2 / 24.6 / 23.1 / 26.1.
//   pair    from 65 tokens on where it is estimated to be faster.  The estimates (microseconds; fixed part, then the time
//           of a 128-column block per wave of tiles, or the bytes read by the SMs) fit 128 x 4096 x 4096 (split 9.0, pair
//           9.2), 77 x 12288 x 4096 (14.7, 25), 128 x 4096 x 24576 (30.8, 24.2), 200 x 4096 x 4096 (11.3, 9.5), 512 x 4096 x
//           24576 (pair of 128 tokens 50, of 256 44.6) and 512 x 4096 x 4096 (11.6, 15.5) on the right side.
Plan plan(int n_rows, int kb, int n_tok) {
    Plan best = {n_tok <= 16 ? 16 : n_tok <= 32 ? 32 : 64, 1};
    const long long row_tiles = (n_rows + 127) / 128, tiles = row_tiles * ((n_tok + best.ntok - 1) / best.ntok);
    for (int s = 2; s <= MAX_SPLIT && 2 * s <= kb; s++)
        if (tiles <= g_clusters[s]) best.split = s;
    if (n_tok <= 64) return best;
    const double hbm = ((double)row_tiles * kb * W_TILE + 4.0 * n_rows * n_tok) / 6.0e6;
    double best_t = 5.0 + std::max((double)tiles * kb * (W_TILE + 64 * 128) / 13.0e6, hbm);
    for (int nt = 128; nt <= 256; nt *= 2) {
        const long long pairs = (long long)((n_rows + 255) / 256) * ((n_tok + nt - 1) / nt), at_once = g_sm_count / 2;
        const double t = (nt == 128 ? 4.0 : 5.0) + std::max((double)((pairs + at_once - 1) / at_once) * kb * (nt == 128 ? 0.22 : 0.38), hbm);
        if (t < best_t) { best_t = t; best = {nt, 0}; }
    }
    return best;
}

template <int NTOK>
void split_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], dim3 grid, cudaStream_t st) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = SplitCfg<NTOK>::SMEM;
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = grid.x;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
}

template <int NTOK>
int launch_split(const I8Product& p, int split, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    split_config<NTOK>(cfg, attr, dim3(split, (p.n_tok + NTOK - 1) / NTOK, (p.n_rows + 127) / 128), st);
    HB_CUDA(cudaLaunchKernelEx(&cfg, i8_split_kernel<NTOK>, p));
    return 0;
}

template <int NTOK>
int prepare_split() {
    HB_CUDA(cudaFuncSetAttribute(i8_split_kernel<NTOK>, cudaFuncAttributeMaxDynamicSharedMemorySize, SplitCfg<NTOK>::SMEM));
    return 0;
}

template <int NT>
int prepare_pair() {
    HB_CUDA(cudaFuncSetAttribute(i8_pair_kernel<NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg<NT>::SMEM));
    HB_CUDA(cudaFuncSetAttribute(i8_pair_kernel<NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg<NT>::SMEM));
    return 0;
}

}  // namespace

int i8_gemm_prepare(int sm_count) {
    g_sm_count = sm_count;
    int rc;
    if ((rc = prepare_split<16>())) return rc;
    if ((rc = prepare_split<32>())) return rc;
    if ((rc = prepare_split<64>())) return rc;
    for (int s = 2; s <= MAX_SPLIT; s++) {  // (the tiles of 32 and 64 tokens hold as much shared memory)
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[2];
        split_config<16>(cfg, attr, dim3(s, 1, 1), nullptr);
        cfg.numAttrs = 1;
        int n = 0;
        HB_CUDA(cudaOccupancyMaxActiveClusters(&n, i8_split_kernel<16>, &cfg));
        g_clusters[s] = 2 * n;
    }
    if ((rc = prepare_pair<128>())) return rc;
    return prepare_pair<256>();
}

int launch_i8_gemm(const I8Product& p, cudaStream_t st) {
    const Plan pl = plan(p.n_rows, p.kb, p.n_tok);
    if (pl.split == 0) return pl.ntok == 256 ? launch_pair<256>(p, g_sm_count, st) : launch_pair<128>(p, g_sm_count, st);
    switch (pl.ntok) {
        case 16: return launch_split<16>(p, pl.split, st);
        case 32: return launch_split<32>(p, pl.split, st);
        default: return launch_split<64>(p, pl.split, st);
    }
}

const char* i8_gemm_kernel_name(int n_rows, int kb, int n_tok) {
    const Plan pl = plan(n_rows, kb, n_tok);
    if (pl.split == 0) return pl.ntok == 256 ? "i8_tcgen05_pair_n256" : "i8_tcgen05_pair_n128";
    switch (pl.ntok) {
        case 16: return pl.split > 1 ? "i8_tcgen05_n16_split" : "i8_tcgen05_n16";
        case 32: return pl.split > 1 ? "i8_tcgen05_n32_split" : "i8_tcgen05_n32";
        default: return pl.split > 1 ? "i8_tcgen05_n64_split" : "i8_tcgen05_n64";
    }
}

}  // namespace hb200
