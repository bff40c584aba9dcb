// out = residual + act(x . w^T + bias), all float, for batches of rows: both operands are cut into three bfloat16 numbers first,
// v = v1 + v2 2^-8 + v3 2^-16 (each the rounding of what the ones before it leave: three times eight bits hold a float's 24; the powers of two keep
// the small parts out of the subnormal range), and the product runs on pairs of SMs as six of the tensor cores': x1 w1 in one accumulator,
// x1 w2 + x2 w1 in a second (weight 2^-8) and x1 w3 + x2 w2 + x3 w1 in a third (2^-16). What is left out is below 2^-24 of a product.
//
// Cutting is a pass of its own: 4 bytes an element read, 6 written, at what memory does (32,336 x 1000: 47 us, 6.9 TB/s of the 10 bytes, part of them in
// L2). Where a matrix meets several tiles of rows it pays: a product that cuts on its way (linear_f32_tc.cu) spends two thirds of its
// issue slots on that, for every 64 rows anew. 333 x 32003 x 1000 209 us (297 there), 301 x 2301 x 1000 29 (39), 2000 x 4000 x 2000 172 (338).
//
// The tensor core's additions truncate, so few follow one another where it counts: the accumulator of x1 w1 starts anew every 64 elements of
// K (two take turns) and is added to a float in registers; the other two, whose errors weigh 2^-8, run over 512 elements, and their ends lie 256
// apart: while the warps read one, the MMAs of the next block go to the others first.
// Four warps do that, a row and all of the tile's columns (128 at most) a thread. A block's six products take 12 W cycles of the tensor pipe; 2,100 to 2,500
// pass at W = 128 (copies from L2, 72 KB a CTA, take 1,300) and 1,400 at W = 32, where an MMA takes no less than some 55. Stages more than two and
// accumulators more than two change nothing; freeing an accumulator with a release at cluster scope did: 1,100 cycles a block.
//
// Results that are not finite are computed again by plain multiply-adds, so that infinities and NaN come out as they do there.
#include "act_end.cuh"
#include "tma_map.cuh"
#include <type_traits>

IB_DEFINE_LAST_ERROR()

namespace {

using namespace ib::act;

constexpr int BM = 128, BK = 64, UMMA_K = 16, EPILOGUE_WARPS = 4, NUM_THREADS = 64 + 32 * EPILOGUE_WARPS;
constexpr int STAGES = 3, MAX_WIDTH = 128, TMEM_COLS = 512;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = MAX_WIDTH / 2 * BK * 2, STAGE_BYTES = 3 * (A_BYTES + B_BYTES);
constexpr int BARS_BYTES = 256, BLOCK_BYTES = 32 * 16 * 4;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + BARS_BYTES + EPILOGUE_WARPS * BLOCK_BYTES;
constexpr int CHAIN = 8;                          // blocks of 64 elements that the small products' accumulators run over
constexpr int STATUS_TIMEOUT_PRODUCER = 161, STATUS_TIMEOUT_MMA = 162, STATUS_TIMEOUT_EPILOGUE = 163;
static_assert(SMEM_BYTES <= 227 * 1024 && (2 * STAGES + 8) * 8 + 8 <= BARS_BYTES, "shared memory");

// ------------------------------------------------------------------------------------------------ cutting
// Rows of x, then of w, [rows, K] -> three matrices [rows, pitch] one behind the other, zeros behind K. A thread takes 8 elements; bound by the
// bytes it moves.
constexpr int CUT_THREADS = 128;

template <bool VEC>
__global__ void __launch_bounds__(CUT_THREADS)
cut_kernel(const float* __restrict__ x, const float* __restrict__ w, int64_t M, int64_t N, int64_t K, int64_t pitch, bf16* xs, bf16* ws) {
    const int64_t k = (int64_t(blockIdx.y) * CUT_THREADS + threadIdx.x) * 8;
    ib::pdl_wait();
    if (k >= pitch) return;
    const bool of_x = int64_t(blockIdx.x) < M;
    const int64_t row = of_x ? int64_t(blockIdx.x) : int64_t(blockIdx.x) - M, rows = of_x ? M : N;
    const float* from = (of_x ? x : w) + row * K;
    float v[8];
    if (VEC && k + 8 <= K) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(from + k)), b = __ldcs(reinterpret_cast<const float4*>(from + k + 4));
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = k + i < K ? from[k + i] : 0.0f;
    }
    bf16* to = (of_x ? xs : ws) + row * pitch + k;
#pragma unroll
    for (int part = 0; part < 3; part++) {
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const __nv_bfloat162 both = __floats2bfloat162_rn(v[i], v[i + 1]);
            h[i / 2] = *reinterpret_cast<const uint32_t*>(&both);
            v[i] = (v[i] - __low2float(both)) * 256.0f;                        // both operations are exact; an infinity leaves NaN
            v[i + 1] = (v[i + 1] - __high2float(both)) * 256.0f;
        }
        *reinterpret_cast<uint4*>(to + part * rows * pitch) = make_uint4(h[0], h[1], h[2], h[3]);
    }
}

// ------------------------------------------------------------------------------------------------ the product
struct CutParams : EndParams {
    int blocks, width, tiles_m, tiles_n, a_rows;
    int64_t K;
    const float *x, *w;          // for results that are not finite
    int* status;
};

// By a whole warp, 256 elements of K at a time; every lane has the result. Ends where the sum is NaN, which it stays.
__device__ __noinline__ float plain_product(const float* x, const float* w, int64_t K) {
    const int lane = threadIdx.x & 31;
    float s[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
    for (int64_t k = 0; k < K; k += 256) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int64_t at = k + 32 * i + lane;
            if (at < K) s[i] = fmaf(x[at], w[at], s[i]);
        }
        sum = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
        if (__any_sync(0xffffffffu, isnan(sum))) return __int_as_float(0x7fffffff);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

template <int ACT>
__global__ void __launch_bounds__(NUM_THREADS)
cut_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const CutParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + STAGES * STAGE_BYTES;           // full[], empty[], then full and empty of the two first and of the second and third accumulators
    volatile uint32_t* slots = reinterpret_cast<volatile uint32_t*>(base_ptr + STAGES * STAGE_BYTES + (2 * STAGES + 8) * 8);
    // slots[0] = TMEM base address, slots[1] = abort flag (of this CTA)
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int walker = blockIdx.x / 2, walkers = gridDim.x / 2, n_tiles = p.tiles_m * p.tiles_n;
    const int b_rows = p.width / 2, a_bytes = p.a_rows * BK * 2, b_bytes = b_rows * BK * 2;
    // Whether the second (i = 0) or third accumulator starts anew with a block, and whether it ends with it.
    auto starts = [&](int i, int kb) { return kb == 0 || kb % CHAIN == i * (CHAIN / 2); };
    auto ends = [&](int i, int kb) { return kb + 1 == p.blocks || (kb + 1) % CHAIN == i * (CHAIN / 2); };
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
    auto main_full = [&](int b) { return bars + 8u * (2 * STAGES + b); };
    auto main_empty = [&](int b) { return bars + 8u * (2 * STAGES + 2 + b); };
    auto small_full = [&](int b) { return bars + 8u * (2 * STAGES + 4 + b); };
    auto small_empty = [&](int b) { return bars + 8u * (2 * STAGES + 6 + b); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int b = 0; b < 2; b++) {
            mbar_init(main_full(b), 1); mbar_init(main_empty(b), 2 * EPILOGUE_WARPS);
            mbar_init(small_full(b), 1); mbar_init(small_empty(b), 2 * EPILOGUE_WARPS);
        }
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
    cluster_sync();                                               // the other CTA's barriers are initialised
    tc_fence_after();
    const uint32_t tmem_base = slots[0];                          // columns 0, 128: x1 w1; 256: weight 2^-8; 384: 2^-16

    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer (of each CTA)
        if (lane == 0) {
            ib::pdl_wait();
            int it = 0, s = 0;
            uint32_t parity = 1;                                  // of the wait for the slot's use before
            for (int tile = walker; tile < n_tiles && !slots[1]; tile += walkers) {
                const int a_row = ((tile % p.tiles_m) * 2 + int(rank)) * p.a_rows, b_row = (tile / p.tiles_m) * p.width + int(rank) * b_rows;
                for (int kb = 0; kb < p.blocks; kb++, it++) {
                    if (it >= STAGES && !mbar_wait(empty_bar(s), parity)) {
                        atomicExch(p.status, STATUS_TIMEOUT_PRODUCER); slots[1] = 1; break;
                    }
                    if (slots[1]) break;
                    const uint32_t dst = base + s * STAGE_BYTES, bar = map_cluster(full_bar(s), 0u);
                    if (rank == 0) mbar_expect_tx(full_bar(s), uint32_t(6 * (a_bytes + b_bytes)));
#pragma unroll
                    for (int part = 0; part < 3; part++) {
                        load_tile(dst + part * A_BYTES, &tm_a, bar, kb * BK, part * int(p.M) + a_row);
                        load_tile(dst + 3 * A_BYTES + part * B_BYTES, &tm_b, bar, kb * BK, part * int(p.N) + b_row);
                    }
                    if (++s == STAGES) { s = 0; parity ^= 1u; }
                }
            }
            // What another CTA sends here lands before this one ends: the commits that free the last stages, and where a wait ran out the copies
            // of every stage that the first CTA was told of.
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
            const bool leader = elect_one();
            int s = 0, use = 0;                                   // use: of the first accumulators, in turns
            uint32_t parity = 0, used = 0, turn = 0;              // bit i: the second (third) accumulator was used, an odd number of times
            bool ok = true;
            for (int tile = walker; tile < n_tiles && ok; tile += walkers) {
                for (int kb = 0; kb < p.blocks; kb++) {
                    const int b = use & 1;
                    if (use >= 2 && !mbar_wait_each(main_empty(b), ((use >> 1) - 1) & 1)) { ok = false; break; }
                    if (!mbar_wait_each(full_bar(s), parity)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t at = base + s * STAGE_BYTES, d = tmem_base + uint32_t(b * 128);
                    uint64_t x[3], w[3];
#pragma unroll
                    for (int i = 0; i < 3; i++) { x[i] = make_desc(at + i * A_BYTES, 16, 1024); w[i] = make_desc(at + 3 * A_BYTES + i * B_BYTES, 16, 1024); }
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; k++) umma_pair(d, x[0] + uint64_t(2 * k), w[0] + uint64_t(2 * k), idesc, k > 0);
                        commit_pair(main_full(b), 3);
                    }
                    __syncwarp();
                    // The accumulator that ends with this block comes first, the one that starts anew last: it may still be read.
                    const int order = (starts(0, kb) && kb > 0) || (ends(1, kb) && !ends(0, kb));
                    auto add_small = [&](auto which) {
                        constexpr int i = decltype(which)::value;
                        const bool first = starts(i, kb);
                        if (first && (used >> i & 1)) {
                            if (!mbar_wait_each(small_empty(i), (turn >> i & 1) ^ 1)) { ok = false; return; }
                            tc_fence_after();
                        }
                        if (leader) {
                            const uint32_t e = tmem_base + uint32_t(256 + i * 128);
#pragma unroll
                            for (int k = 0; k < BK / UMMA_K; k++) {
                                const uint64_t q = uint64_t(2 * k);
                                umma_pair(e, x[0] + q, w[1 + i] + q, idesc, (!first || k > 0) ? 1u : 0u);
                                umma_pair(e, x[1 + i] + q, w[0] + q, idesc, 1u);
                                if (i == 1) umma_pair(e, x[1] + q, w[1] + q, idesc, 1u);
                            }
                            if (ends(i, kb)) commit_pair(small_full(i), 3);
                        }
                        __syncwarp();
                        if (ends(i, kb)) { used |= 1u << i; turn ^= 1u << i; }
                    };
                    using std::integral_constant;
                    if (order) { add_small(integral_constant<int, 1>{}); if (ok) add_small(integral_constant<int, 0>{}); }
                    else { add_small(integral_constant<int, 0>{}); if (ok) add_small(integral_constant<int, 1>{}); }
                    if (!ok) break;
                    if (leader) commit_pair(empty_bar(s), 3);
                    __syncwarp();
                    use++;
                    if (++s == STAGES) { s = 0; parity ^= 1u; }
                }
            }
            ib::pdl_launch_dependents();
            // (the other CTA's warps have said of each accumulator that they have read it)
            ok = ok && ib::last_uses(use, 2, [&](int b, uint32_t phase) { return mbar_wait_each(main_empty(b), phase); });
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (ok && (used >> i & 1)) ok = mbar_wait_each(small_empty(i), (turn >> i & 1) ^ 1);
            if (!ok && lane == 0) { atomicExch(p.status, STATUS_TIMEOUT_MMA); slots[1] = 1; }
        } else {
            ib::pdl_launch_dependents();
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- epilogue: a row and the tile's columns a thread
        const int quad = warp & 3;
        uint8_t* block = base_ptr + STAGES * STAGE_BYTES + BARS_BYTES + (warp - 2) * BLOCK_BYTES;
        const uint32_t lanes = tmem_base + (uint32_t(quad * 32) << 16);
        ib::pdl_wait();
        int use = 0;
        uint32_t turn = 0;
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = __all_sync(0xffffffffu, !slots[1]);
            if (ok && !mbar_wait_warp(bar, parity)) { atomicExch(p.status, STATUS_TIMEOUT_EPILOGUE); slots[1] = 1; ok = false; }
            tc_fence_after();
            return ok;
        };
        float acc[MAX_WIDTH];
        auto add = [&](uint32_t columns, float weight) {
#pragma unroll
            for (int c = 0; c < MAX_WIDTH; c += 16) {
                if (c < p.width) {
                    float v[16];
                    tmem_get16(columns + uint32_t(c), v);
#pragma unroll
                    for (int j = 0; j < 16; j++) acc[c + j] = fmaf(v[j], weight, acc[c + j]);
                }
            }
        };
        auto release = [&](uint32_t bar) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_cluster(bar, 0u));
        };
        for (int tile = walker; tile < n_tiles && ok; tile += walkers) {
            const int64_t m_cta = int64_t((tile % p.tiles_m) * 2 + int(rank)) * p.a_rows, m0 = m_cta + quad * 32, m_end = min(p.M, m_cta + p.a_rows);
            const int64_t n0 = int64_t(tile / p.tiles_m) * p.width;
            TileEnd end;
            end.open(p, m0, m_end, n0);
#pragma unroll
            for (int c = 0; c < MAX_WIDTH; c++) acc[c] = 0.0f;
            for (int kb = 0; kb < p.blocks; kb++, use++) {
                if (!wait(main_full(use & 1), (use >> 1) & 1)) break;
                add(lanes + uint32_t((use & 1) * 128), 1.0f);
                release(main_empty(use & 1));
#pragma unroll 1
                for (int i = 0; i < 2 && ok; i++) {
                    if (!ends(i, kb)) continue;
                    if (!wait(small_full(i), turn >> i & 1)) break;
                    add(lanes + uint32_t(256 + i * 128), i == 0 ? 0x1p-8f : 0x1p-16f);
                    release(small_empty(i));
                    turn ^= 1u << i;
                }
                if (!ok) break;
            }
            if (!ok) break;
            const int64_t m = m0 + lane;
#pragma unroll
            for (int c = 0; c < MAX_WIDTH; c += 16) {
                if (c < p.width) {
                    float v[16];
                    bool fine = true;
#pragma unroll
                    for (int j = 0; j < 16; j++) { v[j] = acc[c + j]; fine = fine && isfinite(v[j]); }
                    if (__any_sync(0xffffffffu, !fine && m < m_end)) {
#pragma unroll 1
                        for (int j = 0; j < 16 && n0 + c + j < p.N; j++) {
                            float z = 0.0f;
#pragma unroll
                            for (int i = 0; i < 16; i++) z = i == j ? v[i] : z;
                            for (uint32_t bad = __ballot_sync(0xffffffffu, !isfinite(z) && m < m_end); bad; bad &= bad - 1) {
                                const int row = __ffs(int(bad)) - 1;
                                const float again = plain_product(p.x + (m0 + row) * p.K, p.w + (n0 + c + j) * p.K, p.K);
                                if (lane == row) z = again;
                            }
#pragma unroll
                            for (int i = 0; i < 16; i++) v[i] = i == j ? z : v[i];
                        }
                    }
                    __syncwarp();
                    end.block<ACT, float>(p, block, c, v, c + 16 < p.width);
                }
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    // Neither CTA's shared memory is needed by the other any more: what was sent to this one's barriers has been waited for above. Where a wait ran out
    // that is not so, and what was sent before is ordered by the barrier itself.
    if (slots[1]) cluster_sync();
    else cluster_meet();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(uint32_t(TMEM_COLS)) : "memory");
    }
}

template <int ACT>
int launch_cut(const CUtensorMap& ma, const CUtensorMap& mb, const CutParams& p, int sms, cudaStream_t stream) {
    static ib::PerDevice allowed, fit;
    if (const int rc = ib::allow_smem(allowed, "linear_f32_cut", cut_pair_kernel<ACT>, SMEM_BYTES)) return rc;
    const int room = fit.get(ib::current_device(), [&] {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(sms & ~1));
        cfg.blockDim = dim3(NUM_THREADS);
        cfg.dynamicSmemBytes = SMEM_BYTES;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, cut_pair_kernel<ACT>, &cfg);
        return e != cudaSuccess ? 0 : clusters < sms / 2 ? clusters : sms / 2;
    });
    if (room < 1) return ib::fail(IB_ERR_CUDA, "linear_f32_cut: no room for a pair of CTAs");
    const int tiles = p.tiles_m * p.tiles_n;
    return ib::launch("linear_f32_cut", cut_pair_kernel<ACT>, dim3(unsigned(2 * (tiles < room ? tiles : room))), dim3(NUM_THREADS), size_t(SMEM_BYTES), stream, 2u, ma, mb, p);
}

}  // namespace

// Width of a tile (32, 64, 96, 128), bytes of scratch, estimated ns. The width with the least of a pair's tiles x (blocks x (560 + 5.2 W) + 20 W);
// 11,000 more and 10 bytes an element to cut at 6 TB/s. Measured, 333 x 32003 x 1000 at 32, 64, 96, 128 columns 420, 276, 238, 209 us;
// 301 x 2301 x 1000 41, 28.7, 30.7, 34.8; 257 x 5000 x 3000 207, 151, 122, 135.
IB_EXPORT int ib_linear_f32_cut_plan(int64_t M, int64_t N, int64_t K, int sms, int* width, int64_t* scratch, int64_t* ns) {
    if (M <= 0 || N <= 0 || K <= 0) return ib::fail(IB_ERR_ARG, "linear_f32_cut: sizes must be positive");
    // (K: a tile whose results are all computed again takes 4096 plain products a warp, 137 ms at 16,384 on all SMs at once, while the issuer waits about a second)
    if (M > 600000000 || N > 600000000 || K > 16384 || sms < 2) return ib::fail(IB_ERR_ARG, "linear_f32_cut: a size is too large");
    const int64_t tm = (M + 2 * BM - 1) / (2 * BM), blocks = (K + BK - 1) / BK, pitch = (K + 7) / 8 * 8;
    int64_t least = -1;
    for (int w : {128, 96, 64, 32}) {
        const int64_t tiles = tm * ((N + w - 1) / w);
        if (tiles >= (1LL << 28)) continue;
        const int64_t cost = (tiles + sms / 2 - 1) / (sms / 2) * (blocks * (560 + 52 * w / 10) + 20 * w);
        if (least < 0 || cost < least) { least = cost; *width = w; }
    }
    if (least < 0) return ib::fail(IB_ERR_ARG, "linear_f32_cut: too many tiles");
    *scratch = 6 * (M + N) * pitch;
    *ns = least + 11000 + *scratch / 3600;
    return IB_OK;
}

// residual may be out. scratch: the plan's bytes, 16-byte aligned, this call's own until it has run.
IB_EXPORT int ib_linear_f32_cut(const float* x, const float* w, const float* bias, const float* residual, float* out, int64_t M, int64_t N, int64_t K,
                                int act, int width, void* scratch, int sms, int* status, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return IB_OK;
    int planned = 0;
    int64_t bytes = 0, ns = 0;
    if (const int rc = ib_linear_f32_cut_plan(M, N, K, sms, &planned, &bytes, &ns)) return rc;
    if (act < 0 || act >= ib::score::ACTIVATIONS) return ib::fail(IB_ERR_ARG, "linear_f32_cut: unknown activation %d", act);
    if (width != 32 && width != 64 && width != 96 && width != 128) return ib::fail(IB_ERR_ARG, "linear_f32_cut: tiles of 32, 64, 96 or 128 columns");
    if (!status || !scratch || (uintptr_t(scratch) & 15)) return ib::fail(IB_ERR_ARG, "linear_f32_cut: a status word and 16-byte aligned scratch are required");
    const int64_t pitch = (K + 7) / 8 * 8;
    bf16 *xs = static_cast<bf16*>(scratch), *ws = xs + 3 * M * pitch;
    const dim3 grid{unsigned(M + N), unsigned((pitch / 8 + CUT_THREADS - 1) / CUT_THREADS)};
    const bool vec = K % 4 == 0 && ((uintptr_t(x) | uintptr_t(w)) & 15) == 0;
    int rc = vec ? ib::launch("cut", cut_kernel<true>, grid, dim3(CUT_THREADS), 0, stream, 1u, x, w, M, N, K, pitch, xs, ws)
                 : ib::launch("cut", cut_kernel<false>, grid, dim3(CUT_THREADS), 0, stream, 1u, x, w, M, N, K, pitch, xs, ws);
    if (rc) return rc;
    CutParams p = {};
    p.M = M; p.N = N; p.K = K;
    p.act = act; p.vec = columns_in_fours(N, out, residual, true);
    p.bias = bias; p.residual = residual; p.out = out; p.status = status;
    p.x = x; p.w = w;
    p.blocks = int((K + BK - 1) / BK);
    p.width = width;
    p.tiles_m = int((M + 2 * BM - 1) / (2 * BM));
    p.tiles_n = int((N + width - 1) / width);
    p.a_rows = int(((M + 2 * p.tiles_m - 1) / (2 * p.tiles_m) + 7) / 8 * 8);
    CUtensorMap ma, mb;
    rc = ib::get_map(xs, 3 * M, pitch, p.a_rows, &ma);
    if (rc) return rc;
    rc = ib::get_map(ws, 3 * N, pitch, width / 2, &mb);
    if (rc) return rc;
    switch (act) {
        case ib::score::NONE: return launch_cut<ib::score::NONE>(ma, mb, p, sms, stream);
        case ib::score::RELU: return launch_cut<ib::score::RELU>(ma, mb, p, sms, stream);
        case ib::score::RELU_SQUARED: return launch_cut<ib::score::RELU_SQUARED>(ma, mb, p, sms, stream);
        case ib::score::GELU_TANH: return launch_cut<ib::score::GELU_TANH>(ma, mb, p, sms, stream);
        case ib::score::GELU: return launch_cut<ib::score::GELU>(ma, mb, p, sms, stream);
        default: return launch_cut<ib::score::SILU>(ma, mb, p, sms, stream);
    }
}
