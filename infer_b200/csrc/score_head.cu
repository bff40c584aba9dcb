// Log probabilities straight from the rows in front of a head: for each row x of [T, H] and the head's matrix w [V, H], both bfloat16, the
// logits z = x . w^T exist in tensor memory only. Each tile of them is folded into its rows' running statistics (maximum m,
// S = sum exp(l - m), D = sum exp(l - m) (l - m), the best `top` of z), which is all that logprob, entropy and alternatives need.
//
// The product's structure is that of the framework's others on pairs of SMs (two CTAs on 256 rows x W columns with
// tcgen05.mma.cta_group::2, each loading its 128 rows and half of the columns' rows by TMA; two accumulators in tensor memory, so that the
// epilogue of one tile runs under the next one's MMAs), or for up to 128 rows a CTA by itself on 128 x W. A thread of the epilogue owns a
// row: its statistics stay in registers while its CTA walks through every chunks-th tile (a chunk of the vocabulary; with neighbouring
// tiles a chunk all CTAs' requests lay the same distance apart: 64 rows x 1536 against 151,936 77 us, so 74; 48 rows x 1024 72 and 53), and
// leave them once, at the chunk's end. A second, small kernel joins the chunks of a row in ascending order.
//
// Which chunk a CTA works on: unit u = (row block u mod R, chunk u / R), so that CTAs that run together read the same columns' rows of w,
// which then come from HBM once and from L2 R times.
//
// A logit is one chain over H in the tensor core's accumulator, whose additions truncate: off by 4e-6 in norm at H = 3,584, by 1e-5 at 8,960 (for few rows
// the matrix is streamed, with shorter chains: the last digits depend on the number of rows).
//
// Bound by the MMAs (2 T H V operations) from about 256 rows on, below by the bytes of w. The epilogue needs 7 instructions an element and
// an exponential (a warp's 32 take 8 cycles of the special function unit): 256 columns of 128 rows about 2,500 cycles, while a tile's MMAs
// take 8 H (12,288 at H = 1536). Measured against 151,936 x 1536 (bfloat16, in a graph): 17 to 128 rows 74 to 80 us (6.3 TB/s), 2,048 rows 557 us
// (1,713 TFLOP/s; 640 to 670 back to back, at the power limit), 622 with 5 alternatives and 714 with 20 in a row of calls at that limit.
#include "common.cuh"
#include "score.cuh"
#include "tc_ops.cuh"
#include "tma_map.cuh"

IB_DEFINE_LAST_ERROR()

namespace {

using namespace ib::tc;
using ib::score::Stats;

constexpr int BM = 128, BK = 64, UMMA_K = 16, NUM_THREADS = 192;
constexpr int A_BYTES = BM * BK * 2, MAX_WIDTH = 256, TMEM_COLS = 512;
constexpr int MAX_TOP = ib::score::MAX_TOP;
constexpr int STATUS_TIMEOUT_PRODUCER = 141, STATUS_TIMEOUT_MMA = 142, STATUS_TIMEOUT_EPILOGUE = 143;

__device__ __forceinline__ void fence_barrier_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t map_cluster(uint32_t local_smem, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_smem), "r"(rank));
    return remote;
}
// Says that tensor memory was read (the reads were awaited, and fenced): no other memory is handed over, so nothing is released. With a release at
// cluster scope this took 1,100 cycles, in which the warp waits for all it has under way. The issuer waits for all but an accumulator's last; those are
// ordered by the last barrier of the pair, which releases and acquires.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t remote_bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_bar) : "memory");
}
__device__ __forceinline__ uint64_t policy_evict_first() {
    uint64_t pol;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));
    return pol;
}
// A copy into this CTA's shared memory; for a pair it is counted on a barrier of either CTA. `once`: the tile leaves L2 first.
template <int CG> __device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, bool once, uint64_t policy) {
    if constexpr (CG == 1) {
        if (once) asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
                               ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "l"(policy) : "memory");
        else tma_load_2d(dst, map, bar, x, y);
    } else {
        if (once) asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
                               ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "l"(policy) : "memory");
        else asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                          ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    }
}
template <int CG> __device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1) umma_f16(d, a, b, idesc, accumulate);
    else asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives on the barrier (for a pair: at this place in both CTAs) once every MMA issued so far has finished.
template <int CG> __device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (CG == 1) umma_commit(bar);
    else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(uint16_t(3)) : "memory");
}
// 32 columns of this thread's lane, awaited in the same statement: no use of a register can come before.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* r) {
    uint32_t u[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
          "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]),
          "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]),
          "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(taddr) : "memory");
#pragma unroll
    for (int j = 0; j < 32; j++) r[j] = __uint_as_float(u[j]);
}

// A stage of the operand ring: two k-blocks for a pair, one for a CTA by itself.
template <int CG> struct Ring {
    static constexpr int KPS = CG == 2 ? 2 : 1, STAGES = CG == 2 ? 3 : 4;
    static constexpr int B_BYTES = MAX_WIDTH / CG * BK * 2;
    static constexpr int STAGE_BYTES = KPS * (A_BYTES + B_BYTES), SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256;
};

// The best N of what a row has seen, by falling value; among equal ones the earlier (lower id) first.
template <int N> struct Best {
    float v[N];
    int id[N];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; i++) { v[i] = -INFINITY; id[i] = -1; }
    }
    __device__ __forceinline__ bool wants(float z) const { return z > v[N - 1]; }
    __device__ __forceinline__ void put(bool mine, float z, int n) { // mine: wants(z); among equal values ids come in ascending order
        bool above = mine;                                            // z > v[i]
#pragma unroll
        for (int i = N - 1; i > 0; i--) {
            const bool next = mine && z > v[i - 1];
            v[i] = next ? v[i - 1] : (above ? z : v[i]);
            id[i] = next ? id[i - 1] : (above ? n : id[i]);
            above = next;
        }
        v[0] = above ? z : v[0];
        id[0] = above ? n : id[0];
    }
    // Takes what it wants of 32 neighbouring columns, the largest first (z is used up). One branch for the warp and a round for as many columns as
    // a lane wants: with a branch for each column and lane a single warp on its scheduler waited for most of its time.
    // (`row`: whether the lane has a row; others hold whatever shared memory held, which would keep the warp.)
    __device__ __forceinline__ void take(float (&z)[32], float top, int n0, bool row) {
        for (;; top = ib::score::largest_of<32>(z)) {
            const bool mine = row && wants(top);
            if (!__any_sync(0xffffffffu, mine)) return;
            int at = 0;
#pragma unroll
            for (int j = 31; j >= 0; j--) at = z[j] == top ? j : at;
            put(mine, top, n0 + at);
#pragma unroll
            for (int j = 0; j < 32; j++) z[j] = at == j ? -INFINITY : z[j];
        }
    }
};
template <> struct Best<0> {
    __device__ __forceinline__ void clear() {}
    __device__ __forceinline__ void take(float (&)[32], float, int, bool) {}
};

struct HeadParams {
    int64_t T, V;
    int n_kb, width, tiles_n, chunks, row_blocks;
    int a_rows;                  // rows of a CTA, up to 128: dealt out evenly, so that hardly a copy reaches behind the last row (such rows are not only
                                 // zeros to write: 17 rows in boxes of 128 took 122 us where boxes of 24 take 74; what lies in shared memory
                                 // behind the loaded rows goes into sums that nobody reads)
    int weights_once;            // the matrix is read once: its tiles leave L2 first
    float scale, cap;
    const int* tokens;           // [T] or null
    float4* stats;               // [chunks, T]: m, s, d
    unsigned long long* lists;   // [chunks, T, N] keys
    float* at;                   // [T]: z of the row's token, written where that is a token
    int* status;
};

template <int CG, int N>
__global__ void __launch_bounds__(NUM_THREADS)
head_logprobs_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const HeadParams p) {
    using R = Ring<CG>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
    constexpr int S = R::STAGES, KPS = R::KPS;
    const uint32_t bars = base + S * R::STAGE_BYTES;            // full[S], empty[S], acc_full[2], acc_empty[2]
    volatile uint32_t* slots = reinterpret_cast<volatile uint32_t*>(base_ptr + S * R::STAGE_BYTES + (2 * S + 4) * 8);
    // slots[0] = TMEM base address, slots[1] = abort flag (of this CTA)
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;
    const int walker = blockIdx.x / CG, walkers = gridDim.x / CG, units = p.row_blocks * p.chunks;
    const int n_kb = p.n_kb, b_rows = p.width / CG, a_bytes = p.a_rows * BK * 2, b_bytes = b_rows * BK * 2;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S + s); };
    auto acc_full_bar = [&](int b) { return bars + 8u * (2 * S + b); };
    auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * S + 2 + b); };
    // CTAs of different chunks go through K from different places on, or all SMs would ask the same few L2 slices for x at a time
    auto first_kb = [&](int chunk) { return int(int64_t(chunk) * ((n_kb + KPS - 1) / KPS) / p.chunks) * KPS; };
    auto tiles_of = [&](int chunk) { return (p.tiles_n - chunk + p.chunks - 1) / p.chunks; };         // tiles chunk, chunk + chunks, ...

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int b = 0; b < 2; b++) { mbar_init(acc_full_bar(b), 1); mbar_init(acc_empty_bar(b), 4 * CG); }
        slots[1] = 0;
        fence_barrier_init();
        prefetch_tensormap(&tm_a);
        prefetch_tensormap(&tm_b);
    }
    if (warp == 1) {
        if constexpr (CG == 1) {
            tmem_alloc(smem_u32(const_cast<uint32_t*>(&slots[0])), TMEM_COLS);
            tmem_relinquish();
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                         ::"r"(smem_u32(const_cast<uint32_t*>(&slots[0]))), "r"(uint32_t(TMEM_COLS)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();                      // the other CTA's barriers are initialised
    tc_fence_after();
    const uint32_t tmem_base = slots[0];

    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer (of each CTA)
        if (lane == 0) {
            ib::pdl_wait();
            int it = 0, s = 0;
            uint32_t parity = 1;                                  // of the wait for the slot's use before
            const uint64_t once = policy_evict_first();
            for (int u = walker; u < units && !slots[1]; u += walkers) {
                const int chunk = u / p.row_blocks, a_row = ((u % p.row_blocks) * CG + int(rank)) * p.a_rows;
                for (int tile = chunk; tile < p.tiles_n && !slots[1]; tile += p.chunks) {
                    const int b_row = tile * p.width + int(rank) * b_rows;
                    for (int i = 0, kb = first_kb(chunk); i < n_kb; i += KPS, kb = kb + KPS < n_kb ? kb + KPS : 0, it++) {
                        const int n = min(KPS, n_kb - kb);
                        if (it >= S && !mbar_wait(empty_bar(s), parity)) {
                            atomicExch(p.status, STATUS_TIMEOUT_PRODUCER); slots[1] = 1; break;
                        }
                        if (slots[1]) break;
                        const uint32_t a_dst = base + s * R::STAGE_BYTES, b_dst = a_dst + KPS * A_BYTES;
                        const uint32_t bar = CG == 2 ? map_cluster(full_bar(s), 0u) : full_bar(s);
                        if (rank == 0) mbar_expect_tx(full_bar(s), uint32_t(CG * n * (a_bytes + b_bytes)));
#pragma unroll
                        for (int j = 0; j < KPS; j++) {
                            if (j < n) {
                                load_tile<CG>(a_dst + j * A_BYTES, &tm_a, bar, (kb + j) * BK, a_row, false, once);
                                load_tile<CG>(b_dst + j * R::B_BYTES, &tm_b, bar, (kb + j) * BK, b_row, p.weights_once != 0, once);
                            }
                        }
                        if (++s == S) { s = 0; parity ^= 1u; }
                    }
                }
            }
            // No copy may land after the CTA is gone: the first CTA waits for every stage it was told of. (Without a failure
            // the MMAs, which waited for them, have ended before the last barrier below.)
            if (slots[1] && rank == 0)
                for (int i = it > S ? it - S : 0; i < it; i++) mbar_wait(full_bar(i % S), (i / S) & 1);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            // ---------------------------------------------------------------- MMA issuer (of the pair)
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(p.width >> 3) << 17) | (uint32_t(BM * CG >> 4) << 24);
            const bool leader = elect_one();
            int s = 0, lt = 0;
            uint32_t parity = 0;
            bool ok = true;
            for (int u = walker; u < units && ok; u += walkers) {
                const int chunk = u / p.row_blocks, n_tiles = tiles_of(chunk);
                for (int i = 0; i < n_tiles && ok; i++, lt++) {
                    const int b = lt & 1;
                    if (lt >= 2 && !mbar_wait_each(acc_empty_bar(b), ((lt >> 1) - 1) & 1)) { ok = false; break; }      // it has been drained
                    tc_fence_after();
                    const uint32_t d = tmem_base + uint32_t(b * 256);
                    for (int k0 = 0, kb = first_kb(chunk); k0 < n_kb; k0 += KPS, kb = kb + KPS < n_kb ? kb + KPS : 0) {
                        if (!mbar_wait_each(full_bar(s), parity)) { ok = false; break; }
                        const uint32_t a_addr = base + s * R::STAGE_BYTES;
                        const uint64_t ad = make_desc(a_addr, 16, 1024), bd = make_desc(a_addr + KPS * A_BYTES, 16, 1024);
                        if (leader) {
#pragma unroll
                            for (int k = 0; k < BK / UMMA_K; k++)
                                umma<CG>(d, ad + uint64_t(2 * k), bd + uint64_t(2 * k), idesc, (k0 > 0 || k > 0) ? 1u : 0u);
                            if (KPS == 2 && kb + 1 < n_kb) {
#pragma unroll
                                for (int k = 0; k < BK / UMMA_K; k++)
                                    umma<CG>(d, ad + uint64_t((A_BYTES >> 4) + 2 * k), bd + uint64_t((R::B_BYTES >> 4) + 2 * k), idesc, 1u);
                            }
                            commit<CG>(empty_bar(s));
                            if (k0 + KPS >= n_kb) commit<CG>(acc_full_bar(b));
                        }
                        __syncwarp();
                        if (++s == S) { s = 0; parity ^= 1u; }
                    }
                }
            }
            if (!ok && lane == 0) { atomicExch(p.status, STATUS_TIMEOUT_MMA); slots[1] = 1; }
        }
        ib::pdl_launch_dependents();
    } else {
        // ---------------------------------------------------------------- epilogue (warps 2..5 of each CTA): a thread a row
        const int quad = warp & 3;
        ib::pdl_wait();
        int lt = 0;
        bool ok = true;
        for (int u = walker; u < units && ok; u += walkers) {
            const int chunk = u / p.row_blocks;
            const int64_t row = int64_t((u % p.row_blocks) * CG + int(rank)) * p.a_rows + quad * 32 + lane;
            const bool live = quad * 32 < p.a_rows && row - lane < p.T;                  // (of the warp: some row of it is one)
            const bool mine = quad * 32 + lane < p.a_rows && row < p.T;
            const int token = p.tokens && mine ? p.tokens[row] : -1;
            Stats st;
            st.clear();
            Best<N> best;
            best.clear();
            for (int tile = chunk; tile < p.tiles_n; tile += p.chunks, lt++) {
                const int b = lt & 1;
                ok = __all_sync(0xffffffffu, !slots[1]);
                if (ok && !mbar_wait_warp(acc_full_bar(b), (lt >> 1) & 1)) { atomicExch(p.status, STATUS_TIMEOUT_EPILOGUE); slots[1] = 1; ok = false; }
                if (!ok) break;
                tc_fence_after();
                const uint32_t taddr = tmem_base + (uint32_t(quad * 32) << 16) + uint32_t(b * 256);
                const int n_tile = tile * p.width;
                if (live) {
#pragma unroll 1
                    for (int c = 0; c < p.width; c += 32) {
                        float z[32];
                        __syncwarp();
                        tmem_ld32(taddr + uint32_t(c), z);
                        const int n0 = n_tile + c;
                        if (n0 + 32 > p.V) {
#pragma unroll
                            for (int j = 0; j < 32; j++) z[j] = n0 + j < p.V ? z[j] : -INFINITY;
                        }
                        if (unsigned(token - n0) < 32u && token < p.V) {
                            float found = 0.0f;
#pragma unroll
                            for (int j = 0; j < 32; j++) found = token - n0 == j ? z[j] : found;
                            p.at[row] = found;
                        }
                        if (p.cap > 0.0f) {
                            float l[32];
                            ib::score::cap_logits<32>(l, z, p.scale, p.cap, mine);
                            st.add<32>(l, mine ? ib::score::largest_of<32>(l) : -INFINITY);
                            best.take(z, ib::score::largest_of<32>(z), n0, mine);
                        } else {
                            const float top = ib::score::largest_of<32>(z);
                            st.add<32>(z, mine ? top : -INFINITY, p.scale);
                            best.take(z, top, n0, mine);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (CG == 2) mbar_arrive_cluster(map_cluster(acc_empty_bar(b), 0u));
                    else mbar_arrive(acc_empty_bar(b));
                }
            }
            if (ok && mine) {
                const int64_t at = int64_t(chunk) * p.T + row;
                p.stats[at] = make_float4(st.m, st.s, st.d, 0.0f);
                if constexpr (N > 0) {
#pragma unroll
                    for (int i = 0; i < N; i++) p.lists[at * N + i] = best.id[i] < 0 ? 0 : ib::score::key(best.v[i], uint32_t(best.id[i]));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();               // neither CTA's shared memory is needed by the other any more
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CG == 1) tmem_dealloc(tmem_base, TMEM_COLS);
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(uint32_t(TMEM_COLS)) : "memory");
    }
}

// ------------------------------------------------------------------------------------------------ joining the chunks
// A block a row. The chunks' statistics are joined by one warp. Of the chunks' sorted lists only keys that reach a lower bound of the row's
// top-th best are compared: the best of the lists' last keys, or, with at least `top` lists, the top-th of their first keys (then
// at most `top` lists hold such keys). Every survivor counts those that beat it.
constexpr int JOIN_THREADS = 128;

struct JoinParams {
    int64_t T, V;
    int chunks, n, top;          // n: keys of a list (>= top)
    float scale, cap;
    const int* tokens;
    const float4* stats;
    const unsigned long long* lists;
    const float* at;
    float* logprob;
    float* entropy;
    int* top_ids;
    float* top_logprobs;
    int* status;
};

// How many of n keys in shared memory are above k.
__device__ __forceinline__ int beaten_by(const unsigned long long* keys, int n, unsigned long long k) {
    int above = 0, j = 0;
    for (; j + 8 <= n; j += 8) {
#pragma unroll
        for (int e = 0; e < 8; e++) above += keys[j + e] > k;
    }
    for (; j < n; j++) above += keys[j] > k;
    return above;
}

__global__ void __launch_bounds__(JOIN_THREADS)
join_chunks_kernel(const JoinParams p) {
    extern __shared__ __align__(16) unsigned char join_mem[];
    float4* stats = reinterpret_cast<float4*>(join_mem);               // [chunks]
    unsigned long long* heads = reinterpret_cast<unsigned long long*>(stats + p.chunks);        // [chunks] first keys
    unsigned long long* found = heads + p.chunks;                       // the keys that are compared
    __shared__ unsigned long long bound;
    __shared__ int n_found, n_chosen, chosen[MAX_TOP];
    __shared__ Stats total;
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) { bound = 1; n_found = n_chosen = 0; }
    ib::pdl_wait();
    ib::pdl_launch_dependents();
    auto list = [&](int c) { return p.lists + (int64_t(c) * p.T + row) * p.n; };
    const int token = p.tokens && warp == 0 ? p.tokens[row] : -1;
    const float at = token >= 0 && token < p.V ? p.at[row] : 0.0f;
    for (int c = threadIdx.x; c < p.chunks; c += JOIN_THREADS) {        // (everything that is read at first, in one trip to L2)
        stats[c] = p.stats[int64_t(c) * p.T + row];
        if (p.top) heads[c] = list(c)[0];
    }
    unsigned long long lasts = 1;
    if (p.top && p.chunks < p.top && warp == 0) for (int c = lane; c < p.chunks; c += 32) lasts = max(lasts, list(c)[p.top - 1]);
    __syncthreads();
    if (warp == 0) {
        float m = -INFINITY;
        for (int c = lane; c < p.chunks; c += 32) m = fmaxf(m, stats[c].x);
        m = ib::warp_max(m);
        Stats st{m, 0.0f, 0.0f};
        for (int c = lane; c < p.chunks; c += 32) {
            Stats o{stats[c].x, stats[c].y, stats[c].z};
            o.raise(m);
            st.s += o.s;
            st.d += o.d;
        }
        st.s = ib::warp_sum(st.s);
        st.d = ib::warp_sum(st.d);
        if (lane == 0) {
            total = st;
            ib::score::finish(st, token, at, p.scale, p.cap, p.V, p.logprob + row, p.entropy + row, p.status);
        }
    }
    if (p.top == 0) return;
    if (p.chunks >= p.top) {
        for (int c = threadIdx.x; c < p.chunks; c += JOIN_THREADS) {
            const unsigned long long k = heads[c];
            if (k != 0 && beaten_by(heads, p.chunks, k) == p.top - 1) bound = k;
        }
    } else if (warp == 0) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) lasts = max(lasts, __shfl_xor_sync(0xffffffffu, lasts, o));
        if (lane == 0) bound = lasts;
    }
    __syncthreads();
    const unsigned long long least = bound;
    // (at most `top` lists: where there are more, as many as have a first key that reaches the top-th of them. Where a wait of the kernel before ran out lists
    // hold anything, the same key many times too: no more than `top` are taken.)
    for (int c = threadIdx.x; c < p.chunks; c += JOIN_THREADS) {
        if (heads[c] >= least) {
            const int at = atomicAdd(&n_chosen, 1);
            if (at < p.top) chosen[at] = c;
        }
    }
    __syncthreads();
    const int n_keys = min(n_chosen, p.top) * p.top;
    constexpr int EACH = (MAX_TOP * MAX_TOP + JOIN_THREADS - 1) / JOIN_THREADS;
    unsigned long long key[EACH];                                       // (requested together, looked at afterwards)
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int i = threadIdx.x + e * JOIN_THREADS, c = i / p.top;
        key[e] = i < n_keys ? list(chosen[c])[i - c * p.top] : 0;
    }
#pragma unroll
    for (int e = 0; e < EACH; e++)
        if (key[e] >= least) found[atomicAdd(&n_found, 1)] = key[e];
    __syncthreads();
    const int n = n_found;
    const Stats st = total;
    for (int i = threadIdx.x; i < n; i += JOIN_THREADS) {
        const unsigned long long k = found[i];
        const int above = beaten_by(found, n, k);
        if (above < p.top) {
            p.top_ids[row * p.top + above] = int(ib::score::key_id(k));
            p.top_logprobs[row * p.top + above] = ib::score::logprob_of(st, ib::score::key_value(k), p.scale, p.cap);
        }
    }
    for (int i = n + threadIdx.x; i < p.top; i += JOIN_THREADS) {
        p.top_ids[row * p.top + i] = -1;
        p.top_logprobs[row * p.top + i] = -INFINITY;
    }
}

int list_size(int top) { return top == 0 ? 0 : top <= 8 ? 8 : MAX_TOP; }

struct Plan { int group, width, tiles, chunks, row_blocks; };

// Pairs of SMs from 129 rows on. Width of a tile and chunks of the vocabulary: what gives the shortest longest walk, where a tile costs its
// columns and 64 more (its operand rows of x), and a unit two tiles' worth beside its tiles (the accumulators' first fill and last drain, the lists).
Plan find_plan(int64_t T, int64_t V, int sms) {
    Plan best = {};
    best.group = T > BM && sms >= 2 ? 2 : 1;
    best.row_blocks = int((T + BM * best.group - 1) / (BM * best.group));
    const int64_t walkers = sms / best.group;
    int64_t least = -1;
    for (int width : {256, 224, 192, 160, 128}) {
        const int64_t tiles = (V + width - 1) / width;
        const int64_t most = (4 * walkers + best.row_blocks - 1) / best.row_blocks;
        for (int64_t c = 1; c <= tiles && c <= (most < 1 ? 1 : most); c++) {
            const int64_t rounds = (best.row_blocks * c + walkers - 1) / walkers;
            const int64_t cost = rounds * ((tiles + c - 1) / c * (width + 64) + 2 * 320);
            if (least < 0 || cost < least) { least = cost; best.width = width; best.tiles = int(tiles); best.chunks = int(c); }
        }
    }
    return best;
}

// (The search takes as long as a launch: plans are kept by sizes.)
Plan make_plan(int64_t T, int64_t V, int sms) {
    struct Kept { int64_t T = 0, V = 0; int sms = 0; Plan plan = {}; };
    static Kept kept[64];
    static std::mutex mu;
    std::lock_guard<std::mutex> lock(mu);
    Kept& k = kept[(uint64_t(T) * 31 + uint64_t(V)) % 64];
    if (k.T != T || k.V != V || k.sms != sms) { k.plan = find_plan(T, V, sms); k.T = T; k.V = V; k.sms = sms; }
    return k.plan;
}

template <int CG, int N>
int launch_head(const CUtensorMap& ma, const CUtensorMap& mb, const HeadParams& p, int sms, cudaStream_t stream) {
    using R = Ring<CG>;
    static ib::PerDevice allowed, fit;
    if (const int rc = ib::allow_smem(allowed, "head_logprobs", head_logprobs_kernel<CG, N>, R::SMEM_BYTES)) return rc;
    int room = sms;
    if (CG == 2) {
        cudaError_t e = cudaSuccess;
        room = fit.get(ib::current_device(), [&] {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(unsigned(sms & ~1));
            cfg.blockDim = dim3(NUM_THREADS);
            cfg.dynamicSmemBytes = R::SMEM_BYTES;
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            int clusters = 0;
            e = cudaOccupancyMaxActiveClusters(&clusters, head_logprobs_kernel<CG, N>, &cfg);
            return e != cudaSuccess ? 0 : clusters < sms / 2 ? clusters : sms / 2;
        });
        if (room < 1) return ib::fail(IB_ERR_CUDA, "head_logprobs: no room for a pair of CTAs: %s", cudaGetErrorString(e));
    }
    const int units = p.row_blocks * p.chunks;
    return ib::launch("head_logprobs", head_logprobs_kernel<CG, N>, dim3(unsigned(CG * (units < room ? units : room))), dim3(NUM_THREADS),
                      size_t(R::SMEM_BYTES), stream, unsigned(CG), ma, mb, p);
}

}  // namespace

// Bytes of scratch that ib_head_logprobs needs for these sizes (0 and an error code if it refuses them).
IB_EXPORT int ib_head_logprobs_scratch(int64_t T, int64_t V, int64_t H, int top, int sm_count, int64_t* bytes) {
    *bytes = 0;
    if (T <= 0 || V <= 0 || H <= 0) return ib::fail(IB_ERR_ARG, "head_logprobs: sizes must be positive");
    if (H % 8) return ib::fail(IB_ERR_ARG, "head_logprobs: rows of %lld bfloat16 do not keep to 16 bytes", (long long)H);
    if (T >= (1LL << 30) || V >= (1LL << 30) || H >= (1LL << 30)) return ib::fail(IB_ERR_ARG, "head_logprobs: a size exceeds 2^30");
    if (top < 0 || top > MAX_TOP) return ib::fail(IB_ERR_ARG, "head_logprobs: 0 to %d alternatives, not %d", MAX_TOP, top);
    if (sm_count < 1) return ib::fail(IB_ERR_ARG, "head_logprobs: the number of SMs is needed");
    const Plan plan = make_plan(T, V, sm_count);
    *bytes = int64_t(plan.chunks) * T * (16 + 8 * list_size(top)) + 4 * T;
    return IB_OK;
}

// x [T, H], w [V, H] bfloat16, 16-byte aligned; tokens int [T] or null; results as of ib_token_logprobs; scratch: ib_head_logprobs_scratch
// bytes, 16-byte aligned, this call's own until it has run; status: raised where a wait runs out; token_status (or null): set to 1 by a token
// outside the vocabulary other than -1.
IB_EXPORT int ib_head_logprobs(const void* x, const void* w, int64_t T, int64_t V, int64_t H, const int* tokens, int top, float scale, float cap,
                               float* logprob, float* entropy, int* top_ids, float* top_logprobs, void* scratch, int sm_count, int* status,
                               int* token_status, cudaStream_t stream) {
    if (T == 0) return IB_OK;
    int64_t bytes = 0;
    if (const int rc = ib_head_logprobs_scratch(T, V, H, top, sm_count, &bytes)) return rc;
    if ((uintptr_t(x) & 15) || (uintptr_t(w) & 15) || (uintptr_t(scratch) & 15)) return ib::fail(IB_ERR_ARG, "head_logprobs: operands and scratch must be 16-byte aligned");
    if (!(scale > 0.0f) || !(cap >= 0.0f)) return ib::fail(IB_ERR_ARG, "head_logprobs: the scale must be positive, the cap not negative");
    if (!status || !scratch || !logprob || !entropy || (top && (!top_ids || !top_logprobs))) return ib::fail(IB_ERR_ARG, "head_logprobs: results, scratch and a status word are needed");
    const Plan plan = make_plan(T, V, sm_count);
    const int n = list_size(top);
    HeadParams p = {};
    p.T = T; p.V = V;
    p.n_kb = int((H + BK - 1) / BK);
    p.width = plan.width; p.tiles_n = plan.tiles; p.chunks = plan.chunks; p.row_blocks = plan.row_blocks;
    p.weights_once = plan.row_blocks == 1;
    const int64_t ctas = int64_t(plan.row_blocks) * plan.group;
    p.a_rows = int(((T + ctas - 1) / ctas + 7) / 8 * 8);
    p.scale = scale; p.cap = cap; p.tokens = tokens; p.status = status;
    char* s = static_cast<char*>(scratch);
    p.stats = reinterpret_cast<float4*>(s); s += int64_t(plan.chunks) * T * 16;
    p.lists = reinterpret_cast<unsigned long long*>(s); s += int64_t(plan.chunks) * T * 8 * n;
    p.at = reinterpret_cast<float*>(s);
    CUtensorMap ma, mb;
    int rc = ib::get_map(x, T, H, p.a_rows, &ma);
    if (rc) return rc;
    rc = ib::get_map(w, V, H, plan.width / plan.group, &mb);
    if (rc) return rc;
    if (plan.group == 1) rc = n == 0 ? launch_head<1, 0>(ma, mb, p, sm_count, stream) : n == 8 ? launch_head<1, 8>(ma, mb, p, sm_count, stream) : launch_head<1, MAX_TOP>(ma, mb, p, sm_count, stream);
    else rc = n == 0 ? launch_head<2, 0>(ma, mb, p, sm_count, stream) : n == 8 ? launch_head<2, 8>(ma, mb, p, sm_count, stream) : launch_head<2, MAX_TOP>(ma, mb, p, sm_count, stream);
    if (rc) return rc;
    const JoinParams j{T, V, plan.chunks, n, top, scale, cap, tokens, p.stats, p.lists, p.at, logprob, entropy, top_ids, top_logprobs, token_status};
    const int lists = plan.chunks < top ? plan.chunks : top;           // lists that may hold a survivor, at most
    const size_t smem = size_t(plan.chunks) * 24 + size_t(lists) * top * 8;
    if (smem > 48 * 1024) return ib::fail(IB_ERR_ARG, "head_logprobs: %d chunks of the vocabulary are more than their join takes", plan.chunks);
    return ib::launch("join_chunks", join_chunks_kernel, dim3(unsigned(T)), dim3(JOIN_THREADS), smem, stream, 1u, j);
}
