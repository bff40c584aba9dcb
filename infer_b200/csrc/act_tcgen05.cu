// out = residual + act(x . w^T + bias) on pairs of SMs, for more than 128 rows and for fewer where that is faster: x [M, K], w [N, K] bfloat16, bias
// and residual float, out float or bfloat16, rounded once.
//
// Two CTAs (a pair) form 256 rows x W columns with tcgen05.mma.cta_group::2: each loads its 128 rows of x and half of the W rows of w by TMA
// into a ring of stages of two k-blocks (64 elements each), the first CTA's MMA warp issues for both, and each keeps the sums of its
// own rows in its tensor memory, in two accumulators that take turns. Eight warps finish the columns (four, a warp on each scheduler, took as long
// for a tile's gelu as the tile's MMAs at K = 1536).
//
// The tensor core's additions into an accumulator truncate, and the error of a long chain has one sign: 1e-5 of the result after 8,960 elements of
// K. Where the result is float (SUMS), an accumulator starts anew every 768 elements (below 1e-6) and the warps add what it holds to sums in
// registers: 128 a thread, which is why a thread has half of a row's columns. The additions run under the next 768 elements' MMAs. A 16-bit result keeps one chain
// (its half step is 2e-3): at 2048 x 18944 x 3584, relu squared, 0.19 % of the results are the neighbour of the correctly rounded one (sums in 32 bits: 0.03 %).
//
// A long K on few tiles is cut into S = 2 or 4 slices, the pairs of a cluster of 2 S CTAs. Each adds up its slice in registers; when all MMAs of
// the cluster are done, every CTA pushes its columns to the CTAs that own them (a quarter or half each, of its own rows) through
// distributed shared memory, into what was the operand ring, and the owners add the slices in ascending order. No scratch in global memory, no
// counters, nothing that two calls could share.
//
// Bound by the MMAs, or by the way from L2: a k-block of a pair takes 361 + 1.1 W cycles (measured; the MMAs alone 2 W). us in a graph, gelu_tanh,
// bfloat16 and float results: 2048 x 18944 x 3584 180 (1,545 TFLOP/s) and 237, 2048 x 8960 x 1536 47 and 62, 500 x 1536 x 8960 in four slices 22 and 22,
// 1000 x 1536 x 1536 12.1 and 14.9.
#include "act_end.cuh"
#include "tma_map.cuh"

IB_DEFINE_LAST_ERROR()

namespace {

using namespace ib::act;

constexpr int BM = 128, BK = 64, UMMA_K = 16, EPILOGUE_WARPS = 8, NUM_THREADS = 64 + 32 * EPILOGUE_WARPS;
constexpr int STAGES = 3, MAX_WIDTH = 256, TMEM_COLS = 512;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = MAX_WIDTH / 2 * BK * 2, STAGE_BYTES = 2 * (A_BYTES + B_BYTES);
constexpr int BARS_BYTES = 256, BLOCK_BYTES = 32 * 16 * 4;        // BLOCK: a warp's 32 rows x 16 columns on their way to global memory
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + BARS_BYTES + EPILOGUE_WARPS * BLOCK_BYTES;
constexpr int CHAIN = 12;                         // k-blocks that an accumulator adds up before the registers take over (SUMS)
constexpr int COLS = MAX_WIDTH / 2;               // most columns of a thread
constexpr int STATUS_TIMEOUT_PRODUCER = 151, STATUS_TIMEOUT_MMA = 152, STATUS_TIMEOUT_EPILOGUE = 153;
constexpr int GROUP_BYTES = BM * 16 + 32;         // four columns of a CTA's rows, as slices send them
static_assert(MAX_WIDTH / 4 * GROUP_BYTES <= STAGES * STAGE_BYTES, "the slices' columns lie in the ring");

struct ActParams : EndParams {
    int n_kb, width, tiles_m, tiles_n, slices;
    int a_rows;                  // rows of a CTA, up to 128: dealt out evenly, since copies that reach behind the last row take far longer
    int* status;
};

// S: slices of K (a cluster of 2 S CTAs, one tile); 1: the pairs walk over the tiles. SUMS: sums in registers (always with slices).
// ACT: with sums of whole tiles the finishing code is there once for every 16 of a thread's columns, for one activation (for all of them it did
// not fit the instruction cache: 40,000 cycles a tile, and with the sums moved down in a loop they left the registers: 100,000); -1: any.
template <int S, bool SUMS, int ACT, typename TOut>
__global__ void __launch_bounds__(NUM_THREADS)
act_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const ActParams p) {
    static_assert(S == 1 || SUMS, "slices are added in registers");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + STAGES * STAGE_BYTES;           // full[], empty[], acc_full[2], acc_empty[2]
    volatile uint32_t* slots = reinterpret_cast<volatile uint32_t*>(base_ptr + STAGES * STAGE_BYTES + (2 * STAGES + 4) * 8);
    // slots[0] = TMEM base address, slots[1] = abort flag (of this CTA)
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t crank = cluster_rank(), rank = crank & 1u, lead = crank & ~1u;        // in the cluster, in the pair, the pair's first
    const int slice = int(crank >> 1);
    const int walker = blockIdx.x / (2 * S), walkers = gridDim.x / (2 * S), n_tiles = p.tiles_m * p.tiles_n;
    const int kb0 = int(int64_t(slice) * ((p.n_kb + 1) / 2) / S) * 2, kb1 = min(p.n_kb, int(int64_t(slice + 1) * ((p.n_kb + 1) / 2) / S) * 2);
    const int n_kb = kb1 - kb0, chains = SUMS ? (n_kb + CHAIN - 1) / CHAIN : 1;
    const int b_rows = p.width / 2, a_bytes = p.a_rows * BK * 2, b_bytes = b_rows * BK * 2;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
    auto acc_full_bar = [&](int b) { return bars + 8u * (2 * STAGES + b); };
    auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * STAGES + 2 + b); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int b = 0; b < 2; b++) { mbar_init(acc_full_bar(b), 1); mbar_init(acc_empty_bar(b), 2 * EPILOGUE_WARPS); }
        slots[1] = 0;
        fence_barrier_init();
        prefetch_tensormap(&tm_a);
        prefetch_tensormap(&tm_b);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(const_cast<uint32_t*>(&slots[0]))), "r"(uint32_t(TMEM_COLS)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                               // the other CTAs' barriers are initialised
    tc_fence_after();
    const uint32_t tmem_base = slots[0];

    float acc[SUMS ? COLS : 1];                                   // SUMS: this thread's columns
    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer (of each CTA)
        if (lane == 0) {
            // The first stages' weights set out before the wait: no kernel writes them.
            const int pre = walker < n_tiles ? min(STAGES, (n_kb + 1) / 2) : 0;
            for (int i = 0; i < pre; i++) {
                const int kb = kb0 + 2 * i, n = min(2, kb1 - kb);
                if (rank == 0) mbar_expect_tx(full_bar(i), uint32_t(2 * n * (a_bytes + b_bytes)));
                for (int j = 0; j < n; j++)
                    load_tile(base + i * STAGE_BYTES + 2 * A_BYTES + j * B_BYTES, &tm_b, map_cluster(full_bar(i), lead), (kb + j) * BK,
                              (walker / p.tiles_m) * p.width + int(rank) * b_rows);
            }
            ib::pdl_wait();
            int it = 0, s = 0;
            uint32_t parity = 1;                                  // of the wait for the slot's use before
            for (int tile = walker; tile < n_tiles && !slots[1]; tile += walkers) {
                const int a_row = ((tile % p.tiles_m) * 2 + int(rank)) * p.a_rows, b_row = (tile / p.tiles_m) * p.width + int(rank) * b_rows;
                for (int kb = kb0; kb < kb1; kb += 2, it++) {
                    const int n = min(2, kb1 - kb);
                    if (it >= STAGES && !mbar_wait(empty_bar(s), parity)) {
                        atomicExch(p.status, STATUS_TIMEOUT_PRODUCER); slots[1] = 1; break;
                    }
                    if (slots[1]) break;
                    const uint32_t a_dst = base + s * STAGE_BYTES, b_dst = a_dst + 2 * A_BYTES;
                    const uint32_t bar = map_cluster(full_bar(s), lead);
                    if (rank == 0 && it >= pre) mbar_expect_tx(full_bar(s), uint32_t(2 * n * (a_bytes + b_bytes)));
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        if (j < n) {
                            load_tile(a_dst + j * A_BYTES, &tm_a, bar, (kb + j) * BK, a_row);
                            if (it >= pre) load_tile(b_dst + j * B_BYTES, &tm_b, bar, (kb + j) * BK, b_row);
                        }
                    }
                    if (++s == STAGES) { s = 0; parity ^= 1u; }
                }
            }
            // What another CTA sends here lands before this one ends: the commits that free the last stages, and where a wait ran out the copies
            // of every stage that the first CTA was told of. (Without a failure the MMAs waited for those.)
            if (!slots[1] && !ib::last_uses(it, STAGES, [&](int b, uint32_t phase) { return mbar_wait(empty_bar(b), phase); })) {
                atomicExch(p.status, STATUS_TIMEOUT_PRODUCER); slots[1] = 1;
            }
            if (slots[1] && rank == 0) ib::last_uses(it, STAGES, [&](int b, uint32_t phase) { mbar_wait(full_bar(b), phase); return true; });
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            // ---------------------------------------------------------------- MMA issuer (of the pair)
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(p.width >> 3) << 17) | (uint32_t(2 * BM >> 4) << 24);
            const uint16_t both = uint16_t(3u << lead);
            const bool leader = elect_one();
            int s = 0, use = 0;                                   // use: of the accumulators, in turns
            uint32_t parity = 0;
            bool ok = true;
            for (int tile = walker; tile < n_tiles && ok; tile += walkers) {
                for (int kb = 0; kb < n_kb; kb += 2) {
                    const int b = use & 1;
                    const bool first = SUMS ? kb % CHAIN == 0 : kb == 0, last = kb + 2 >= n_kb || (SUMS && (kb + 2) % CHAIN == 0);
                    if (first) {
                        if (use >= 2 && !mbar_wait_each(acc_empty_bar(b), ((use >> 1) - 1) & 1)) { ok = false; break; }      // both CTAs have drained it
                        tc_fence_after();
                    }
                    if (!mbar_wait_each(full_bar(s), parity)) { ok = false; break; }
                    const uint32_t d = tmem_base + uint32_t(b * 256), a_addr = base + s * STAGE_BYTES;
                    const uint64_t ad = make_desc(a_addr, 16, 1024), bd = make_desc(a_addr + 2 * A_BYTES, 16, 1024);
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; k++)
                            umma_pair(d, ad + uint64_t(2 * k), bd + uint64_t(2 * k), idesc, (!first || k > 0) ? 1u : 0u);
                        if (kb + 1 < n_kb) {
#pragma unroll
                            for (int k = 0; k < BK / UMMA_K; k++)
                                umma_pair(d, ad + uint64_t((A_BYTES >> 4) + 2 * k), bd + uint64_t((B_BYTES >> 4) + 2 * k), idesc, 1u);
                        }
                        commit_pair(empty_bar(s), both);
                        if (last) commit_pair(acc_full_bar(b), both);
                    }
                    __syncwarp();
                    if (last) use++;
                    if (++s == STAGES) { s = 0; parity ^= 1u; }
                }
            }
            ib::pdl_launch_dependents();
            // (the other CTA's warps have said of each accumulator that they have read it)
            ok = ok && ib::last_uses(use, 2, [&](int b, uint32_t phase) { return mbar_wait_each(acc_empty_bar(b), phase); });
            if (!ok && lane == 0) { atomicExch(p.status, STATUS_TIMEOUT_MMA); slots[1] = 1; }
        } else {
            ib::pdl_launch_dependents();
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- epilogue: a row of the CTA and half of the columns a thread
        const int quad = warp & 3, half = (warp - 2) >> 2, cols = p.width / 2, c_first = half * cols;
        uint8_t* block = base_ptr + STAGES * STAGE_BYTES + BARS_BYTES + (warp - 2) * BLOCK_BYTES;
        const uint32_t lanes = tmem_base + (uint32_t(quad * 32) << 16) + uint32_t(c_first);
        ib::pdl_wait();
        int use = 0;
        bool ok = true;
        for (int tile = walker; tile < n_tiles && ok; tile += walkers) {
            const int64_t m_cta = int64_t((tile % p.tiles_m) * 2 + int(rank)) * p.a_rows, m0 = m_cta + quad * 32, m_end = min(p.M, m_cta + p.a_rows), n0 = int64_t(tile / p.tiles_m) * p.width + c_first;
            TileEnd end;
            if (S == 1) end.open(p, m0, m_end, n0);
            if constexpr (SUMS) {
#pragma unroll
                for (int c = 0; c < COLS; c++) acc[c] = 0.0f;
            }
            for (int chain = 0; chain < chains; chain++, use++) {
                const int b = use & 1;
                ok = __all_sync(0xffffffffu, !slots[1]);
                if (ok && !mbar_wait_warp(acc_full_bar(b), (use >> 1) & 1)) { atomicExch(p.status, STATUS_TIMEOUT_EPILOGUE); slots[1] = 1; ok = false; }
                if (!ok) break;
                tc_fence_after();
                if constexpr (SUMS) {
#pragma unroll
                    for (int c = 0; c < COLS; c += 16) {
                        if (c < cols) {
                            float v[16];
                            tmem_get16(lanes + uint32_t(b * 256 + c), v);
#pragma unroll
                            for (int j = 0; j < 16; j++) acc[c + j] += v[j];
                        }
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < cols; c += 16) {
                        float v[16];
                        tmem_get16(lanes + uint32_t(b * 256 + c), v);
                        end.block<ACT, TOut>(p, block, c, v, c + 16 < cols);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(map_cluster(acc_empty_bar(b), lead));
            }
            if (S == 1 && SUMS && ok) {
#pragma unroll
                for (int c = 0; c < COLS; c += 16) {
                    if (c < cols) {
                        float v[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) v[j] = acc[c + j];
                        end.block<ACT, TOut>(p, block, c, v, c + 16 < cols);
                    }
                }
            }
        }
        __syncwarp();
    }
    if constexpr (S > 1) {
        cluster_sync();                                  // every MMA of the cluster is done: the rings are free
        // [slice][group of four columns][row][4] of the columns that this CTA owns: width / S from width / S * slice on (32 bytes behind each
        // group: lanes that read two rows of four groups do not meet in a bank)
        const int own = p.width / S, quad = warp & 3, r = quad * 32 + lane, half = (warp - 2) >> 2, cols = p.width / 2;
        if (warp >= 2 && !slots[1]) {
            int owner = half * cols / own, at = half * cols - owner * own;              // (carried along: no division for each column)
            uint32_t to = map_cluster(base, uint32_t(owner * 2) + rank);
#pragma unroll
            for (int c = 0; c < COLS; c += 4) {
                if (c < cols) {
                    st_cluster_v4(to + uint32_t((slice * (own >> 2) + (at >> 2)) * GROUP_BYTES + r * 16), &acc[c]);
                    at += 4;
                    if (at == own) { at = 0; owner++; if (owner < S) to = map_cluster(base, uint32_t(owner * 2) + rank); }
                }
            }
        }
        // A warp finishes 8 rows x 4 groups of columns at a time: rows 8 (warp - 2) + 64 h on, h = 0, 1, of the columns 16 q on; four q are a batch.
        // What is added to the first two batches is requested before the barrier.
        const int groups = own >> 2, per_h = (groups + 15) >> 4, batches = 2 * per_h;     // (S = 2: up to 4, S = 4: 2)
        const int64_t n0 = int64_t(walker / p.tiles_m) * p.width + own * slice;
        auto rows_of = [&](int k) { return 8 * (warp - 2) + (lane >> 2) + (k >= per_h ? 64 : 0); };
        auto first_of = [&](int k) { return (k >= per_h ? k - per_h : k) * 16 + (lane & 3); };         // group of the batch's first four columns; 4 on: the next
        auto four_of = [&](int k) {
            const int64_t m = int64_t((walker % p.tiles_m) * 2 + int(rank)) * p.a_rows + rows_of(k), n = n0 + 4 * first_of(k);
            Four f{m * p.N + n, 16, int(p.N - n), 16, 0u};
#pragma unroll
            for (int j = 0; j < 4; j++) f.live |= rows_of(k) < p.a_rows && m < p.M && first_of(k) + 4 * j < groups && n + 16 * j < p.N ? 1u << j : 0u;
            return f;
        };
        auto request = [&](int k, float4 (&bias)[4], float4 (&add)[4]) {
            const Four f = four_of(k);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                bias[j] = bias_of(p, f.live >> j & 1 ? n0 + 4 * first_of(k) + 16 * j : p.N);
                add[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            if (p.residual) residual_of(p, f, add);
        };
        float4 bias[2][4], add[2][4];
        if (warp >= 2) { request(0, bias[0], add[0]); request(1, bias[1], add[1]); }
        __syncwarp();
        cluster_sync();                                  // every slice's columns have arrived
        if (warp >= 2 && !slots[1]) {
#pragma unroll
            for (int k = 0; k < (S == 2 ? 4 : 2); k++) {
                if (k >= batches) break;
                const Four f = four_of(k);
                float v[16];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (f.live >> j & 1) {
#pragma unroll
                        for (int o = 0; o < S; o++) {
                            const float4 g = *reinterpret_cast<const float4*>(base_ptr + (o * groups + first_of(k) + 4 * j) * GROUP_BYTES + rows_of(k) * 16);
                            z.x += g.x; z.y += g.y; z.z += g.z; z.w += g.w;
                        }
                    }
                    v[4 * j] = z.x + bias[k & 1][j].x; v[4 * j + 1] = z.y + bias[k & 1][j].y; v[4 * j + 2] = z.z + bias[k & 1][j].z; v[4 * j + 3] = z.w + bias[k & 1][j].w;
                }
                values_of<ACT>(p, v, add[k & 1]);
                store_four<TOut>(p, f, v);
                if (k + 2 < batches) request(k + 2, bias[k & 1], add[k & 1]);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    // No CTA's shared memory is needed by another any more: what was sent to this one's barriers has been waited for above, the slices' columns were at
    // their barrier. Where a wait ran out that is not so, and what was sent before is ordered by the barrier itself.
    if (slots[1]) cluster_sync();
    else cluster_meet();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(uint32_t(TMEM_COLS)) : "memory");
    }
}

// Clusters of 2 S CTAs that run at once (at most one CTA an SM).
template <int S, bool SUMS, int ACT, typename TOut> int clusters_at_once(int sms) {
    static ib::PerDevice allowed, fit;
    if (ib::allow_smem(allowed, "linear_act", act_pair_kernel<S, SUMS, ACT, TOut>, SMEM_BYTES)) return 0;
    return fit.get(ib::current_device(), [&] {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(sms / (2 * S) * (2 * S)));
        cfg.blockDim = dim3(NUM_THREADS);
        cfg.dynamicSmemBytes = SMEM_BYTES;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2 * S; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, act_pair_kernel<S, SUMS, ACT, TOut>, &cfg);
        return e != cudaSuccess ? 0 : clusters < sms / (2 * S) ? clusters : sms / (2 * S);
    });
}

template <int S, bool SUMS, int ACT, typename TOut>
int launch_act(const CUtensorMap& ma, const CUtensorMap& mb, const ActParams& p, int sms, cudaStream_t stream) {
    const int room = clusters_at_once<S, SUMS, ACT, TOut>(sms);
    if (room < 1) return ib::fail(IB_ERR_CUDA, "linear_act: no room for a cluster of %d CTAs", 2 * S);
    const int tiles = p.tiles_m * p.tiles_n;
    return ib::launch("linear_act", act_pair_kernel<S, SUMS, ACT, TOut>, dim3(unsigned(2 * S * (S > 1 || tiles < room ? tiles : room))), dim3(NUM_THREADS),
                      size_t(SMEM_BYTES), stream, unsigned(2 * S), ma, mb, p);
}

template <typename TOut> int launch_any(int slices, bool sums, const CUtensorMap& ma, const CUtensorMap& mb, const ActParams& p, int sms, cudaStream_t stream) {
    if (slices == 4) return launch_act<4, true, -1, TOut>(ma, mb, p, sms, stream);
    if (slices == 2) return launch_act<2, true, -1, TOut>(ma, mb, p, sms, stream);
    if constexpr (sizeof(TOut) == 4) {
        if (sums) switch (p.act) {
            case ib::score::NONE: return launch_act<1, true, ib::score::NONE, TOut>(ma, mb, p, sms, stream);
            case ib::score::RELU: return launch_act<1, true, ib::score::RELU, TOut>(ma, mb, p, sms, stream);
            case ib::score::RELU_SQUARED: return launch_act<1, true, ib::score::RELU_SQUARED, TOut>(ma, mb, p, sms, stream);
            case ib::score::GELU_TANH: return launch_act<1, true, ib::score::GELU_TANH, TOut>(ma, mb, p, sms, stream);
            case ib::score::GELU: return launch_act<1, true, ib::score::GELU, TOut>(ma, mb, p, sms, stream);
            default: return launch_act<1, true, ib::score::SILU, TOut>(ma, mb, p, sms, stream);
        }
    }
    return launch_act<1, false, -1, TOut>(ma, mb, p, sms, stream);
}

}  // namespace

// Width of a tile (32 .. 256, a multiple of 32) and slices of K (1, 2 or 4) for a product; sms: of the device. Cycles that a launch takes: rounds x
// (k-blocks of a slice x (361 + 1.1 width) + what follows the last MMA), with that for a whole tile's epilogue 1,000 + 30 width, for
// slices 13,000 beside their own columns' (two barriers, the push, another start).
IB_EXPORT int ib_linear_act_plan(int64_t M, int64_t N, int64_t K, int sms, int* width, int* slices, int64_t* cycles) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 8) return ib::fail(IB_ERR_ARG, "linear_act: sizes must be positive, K a multiple of 8");
    if (M >= (1LL << 30) || N >= (1LL << 30) || K >= (1LL << 30)) return ib::fail(IB_ERR_ARG, "linear_act: a size exceeds 2^30");
    const int64_t tm = (M + 2 * BM - 1) / (2 * BM), kb = (K + BK - 1) / BK;
    int64_t least = -1;
    for (int s : {1, 2, 4}) {
        if (s > 1 && kb < 8 * s) continue;
        // (clusters of four leave some SMs of a GPC idle, clusters of eight up to a fifth)
        const int64_t room = s == 1 ? sms / 2 : s == 2 ? (sms - sms / 16) / 4 : (sms - sms / 6) / 8;
        if (room < 1) continue;
        for (int w : {256, 224, 192, 160, 128, 96, 64, 32}) {
            const int64_t tiles = tm * ((N + w - 1) / w);
            if (tiles >= (1LL << 28) || (s > 1 && tiles > 2 * room)) continue;
            const int64_t rounds = (tiles + room - 1) / room;
            const int64_t cost = s == 1 ? rounds * kb * (361 + 11 * w / 10) + 1000 + 30 * w : rounds * ((kb + s - 1) / s * (361 + 11 * w / 10) + 13000 + 8 * w / s);
            if (least < 0 || cost < least) { least = cost; *width = w; *slices = s; }
        }
    }
    if (least < 0) return ib::fail(IB_ERR_ARG, "linear_act: too many tiles, or fewer than two SMs");
    // (as many tiles, but no wider than they need to be)
    const int64_t tn = (N + *width - 1) / *width;
    if (cycles) *cycles = least;
    *width = int(((N + tn - 1) / tn + 31) / 32 * 32);
    return IB_OK;
}

// x [M, K], w [N, K] bfloat16 with 16-byte aligned bases, K a multiple of 8; bias float [N] or null; residual float [M, N] or null (may be out); act: an
// activation's number; width and slices from ib_linear_act_plan (or others within its ranges).
IB_EXPORT int ib_linear_act(const void* x, const void* w, const float* bias, const float* residual, void* out, int64_t M, int64_t N, int64_t K,
                            int out_dtype, int act, int width, int slices, int sms, int* status, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return IB_OK;
    if (K <= 0 || K % 8) return ib::fail(IB_ERR_ARG, "linear_act: K = %lld must be a positive multiple of 8", (long long)K);
    if ((uintptr_t(x) & 15) || (uintptr_t(w) & 15)) return ib::fail(IB_ERR_ARG, "linear_act: operand bases must be 16-byte aligned");
    if (act < 0 || act >= ib::score::ACTIVATIONS) return ib::fail(IB_ERR_ARG, "linear_act: unknown activation %d", act);
    if (width < 32 || width > MAX_WIDTH || width % 32 || (slices != 1 && slices != 2 && slices != 4)) return ib::fail(IB_ERR_ARG, "linear_act: tiles of 32 to 256 columns in steps of 32, 1, 2 or 4 slices");
    if (!status || sms < 2) return ib::fail(IB_ERR_ARG, "linear_act: a status word and the number of SMs are required");
    ActParams p = {};
    p.M = M; p.N = N;
    p.n_kb = int((K + BK - 1) / BK);
    if (slices > 1 && p.n_kb < 2 * slices) return ib::fail(IB_ERR_ARG, "linear_act: K = %lld is too short for %d slices", (long long)K, slices);
    const int64_t tm = (M + 2 * BM - 1) / (2 * BM), tn = (N + width - 1) / width;
    if (tm * tn >= (1LL << 28)) return ib::fail(IB_ERR_ARG, "linear_act: too many tiles");
    p.width = width; p.tiles_m = int(tm); p.tiles_n = int(tn); p.slices = slices;
    p.a_rows = int(((M + 2 * tm - 1) / (2 * tm) + 7) / 8 * 8);
    p.act = act; p.bias = bias; p.residual = residual; p.out = out; p.status = status;
    p.vec = columns_in_fours(N, out, residual, out_dtype == IB_F32);
    CUtensorMap ma, mb;
    int rc = ib::get_map(x, M, K, p.a_rows, &ma);
    if (rc) return rc;
    rc = ib::get_map(w, N, K, width / 2, &mb);
    if (rc) return rc;
    if (out_dtype == IB_F32) return launch_any<float>(slices, p.n_kb > CHAIN, ma, mb, p, sms, stream);
    if (out_dtype == IB_BF16) return launch_any<bf16>(slices, false, ma, mb, p, sms, stream);
    return ib::fail(IB_ERR_ARG, "linear_act: unknown output dtype %d", out_dtype);
}
