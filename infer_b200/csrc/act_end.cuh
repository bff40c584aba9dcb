// Shared by the products on pairs of SMs that finish their results themselves (act_tcgen05.cu, linear_f32_cut.cu): the pair's copies and MMAs, and the
// end of a tile: bias, activation, residual, one rounding, coalesced stores.
#pragma once
#include "common.cuh"
#include "last_uses.h"
#include "score.cuh"
#include "tc_ops.cuh"

namespace ib {
namespace act {

using namespace ib::tc;
using bf16 = __nv_bfloat16;

__device__ __forceinline__ void fence_barrier_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same without handing memory over: no thread waits for its stores (3,000 cycles behind a tile's). It orders no arrival on another CTA's barrier either:
// before a CTA may end behind it, each barrier's last uses must have been waited for in the CTA that has it (last_uses).
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
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
// cluster scope this took 1,100 cycles, in which the warp waits for all it has under way. The issuer waits for each of them, the last ones behind its loop.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t remote_bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote_bar) : "memory");
}
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, const float* v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
}
// A copy into this CTA's shared memory, counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t cluster_bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(map), "r"(cluster_bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void umma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives on the barrier at this place in both CTAs of the pair (`mask`: their ranks) once every MMA issued so far has finished.
__device__ __forceinline__ void commit_pair(uint32_t bar, uint16_t mask) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(mask) : "memory");
}
// 16 columns of this thread's lane, awaited in the same statement: no use of a register can come before.
__device__ __forceinline__ void tmem_get16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
#pragma unroll
    for (int j = 0; j < 16; j++) v[j] = __uint_as_float(r[j]);
}

// What the end of a tile needs.
struct EndParams {
    int64_t M, N;
    int act, vec;                // vec: four columns of out (16 or 8 bytes) and residual (16) start on such a boundary
    const float* bias;           // [N] or null
    const float* residual;       // [M, N] or null (may be out)
    void* out;
};
inline int columns_in_fours(int64_t N, const void* out, const float* residual, bool f32) {
    return N % 4 == 0 && (uintptr_t(out) & (f32 ? 15 : 7)) == 0 && (uintptr_t(residual) & 15) == 0;
}

// Four times four neighbouring columns that a lane finishes: number i starts `at` + i step elements into the result, with left - i less columns up to
// the row's end, and is there if bit i of `live` is set.
struct Four {
    int64_t at, step;
    int left, less;
    uint32_t live;
};
__device__ __forceinline__ void residual_of(const EndParams& p, const Four& f, float4 (&add)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        add[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (!(f.live >> i & 1)) continue;
        const float* at = p.residual + f.at + i * f.step;
        if (p.vec) { add[i] = *reinterpret_cast<const float4*>(at); continue; }
        const int left = f.left - i * f.less;
        add[i].x = at[0];
        if (left > 1) add[i].y = at[1];
        if (left > 2) add[i].z = at[2];
        if (left > 3) add[i].w = at[3];
    }
}
__device__ __forceinline__ float4 bias_of(const EndParams& p, int64_t n) {
    float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (!p.bias) return f;
    if (n < p.N) f.x = __ldg(p.bias + n);
    if (n + 1 < p.N) f.y = __ldg(p.bias + n + 1);
    if (n + 2 < p.N) f.z = __ldg(p.bias + n + 2);
    if (n + 3 < p.N) f.w = __ldg(p.bias + n + 3);
    return f;
}
// v[4 i + j] = column j of number i with its bias. ACT < 0: which activation is a parameter of the launch.
template <int ACT>
__device__ __forceinline__ void values_of(const EndParams& p, float (&v)[16], const float4 (&add)[4]) {
    if constexpr (ACT < 0) ib::score::activate_all<16>(v, p.act);
    else {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = ib::score::activate(v[i], ACT);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) { v[4 * i] += add[i].x; v[4 * i + 1] += add[i].y; v[4 * i + 2] += add[i].z; v[4 * i + 3] += add[i].w; }
}
template <typename TOut>
__device__ __forceinline__ void store_four(const EndParams& p, const Four& f, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (!(f.live >> i & 1)) continue;
        const float x = v[4 * i], y = v[4 * i + 1], z = v[4 * i + 2], w = v[4 * i + 3];
        TOut* at = static_cast<TOut*>(p.out) + f.at + i * f.step;
        if (p.vec) {
            if constexpr (sizeof(TOut) == 4) *reinterpret_cast<float4*>(at) = make_float4(x, y, z, w);
            else {
                const __nv_bfloat162 a = __floats2bfloat162_rn(x, y), b = __floats2bfloat162_rn(z, w);
                *reinterpret_cast<uint2*>(at) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
            }
        } else {
            const int left = f.left - i * f.less;
            at[0] = ib::from_f32<TOut>(x);
            if (left > 1) at[1] = ib::from_f32<TOut>(y);
            if (left > 2) at[2] = ib::from_f32<TOut>(z);
            if (left > 3) at[3] = ib::from_f32<TOut>(w);
        }
    }
}

// The columns of a warp's 32 rows of a finished tile, 16 at a time. They pass through the warp's block of shared memory, so that four lanes share
// a row's 64 bytes: with a row a lane, a store of the warp touched 32 lines, and a tile of float results took longer to store than to
// multiply at K = 1536. Units of 16 bytes, those of two rows in a line, are exchanged so that no two lanes meet in a bank. The bias is
// read once a tile and the residual a block ahead: a trip to L2 for each block took 1,300 cycles of its 1,600.
struct TileEnd {
    Four f;                      // of the tile's first 16 columns
    uint32_t rows;
    float4 bias, add[4];         // bias: of columns 4 lane on
    __device__ __forceinline__ void open(const EndParams& p, int64_t m0, int64_t m_end, int64_t n0) {
        const int lane = threadIdx.x & 31, unit = lane & 3;
        const int64_t m = m0 + (lane >> 2);
        f.at = m * p.N + n0 + 4 * unit;
        f.step = 8 * p.N;
        f.left = int(p.N - n0) - 4 * unit;
        f.less = 0;
        rows = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) rows |= m + 8 * i < m_end ? 1u << i : 0u;
        f.live = f.left > 0 ? rows : 0u;
        bias = bias_of(p, n0 + 4 * lane);
#pragma unroll
        for (int i = 0; i < 4; i++) add[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (p.residual) residual_of(p, f, add);
    }
    // v: this lane's row's 16 columns from c on. more: there are 16 others behind them.
    template <int ACT, typename TOut>
    __device__ __forceinline__ void block(const EndParams& p, uint8_t* mem, int c, const float (&v)[16], bool more) {
        const int lane = threadIdx.x & 31, unit = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; i++)
            *reinterpret_cast<float4*>(mem + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        __syncwarp();
        const int from = (c >> 2) + unit;                         // the lane that has these columns' bias
        const float4 b = make_float4(__shfl_sync(0xffffffffu, bias.x, from), __shfl_sync(0xffffffffu, bias.y, from),
                                     __shfl_sync(0xffffffffu, bias.z, from), __shfl_sync(0xffffffffu, bias.w, from));
        float x[16];
        float4 now[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = 8 * i + (lane >> 2);
            const float4 z = *reinterpret_cast<const float4*>(mem + row * 64 + ((unit ^ ((row >> 1) & 3)) << 4));
            x[4 * i] = z.x + b.x; x[4 * i + 1] = z.y + b.y; x[4 * i + 2] = z.z + b.z; x[4 * i + 3] = z.w + b.w;
            now[i] = add[i];
        }
        const Four here = f;
        f.at += 16;
        f.left -= 16;
        f.live = f.left > 0 ? rows : 0u;
        if (p.residual && more) residual_of(p, f, add);
        values_of<ACT>(p, x, now);
        __syncwarp();                                             // the block has been read
        if (sizeof(TOut) == 4 || p.vec) store_four<TOut>(p, here, x);
        else store_columns<TOut>(p, mem, here, x);
    }
    // Rows of 16-bit numbers that do not keep to four columns: the values go back into the block, and sixteen lanes store a row's columns, two rows at
    // a time. (A lane's four columns one by one touch every sector four times: 2000 x 4001 x 512 35 us, this way 26, with 4,000 columns 14.
    // Floats lose by it: 776 x 13581 x 264 on the 32-bit kernel 78 and 91.)
    template <typename TOut>
    __device__ __forceinline__ void store_columns(const EndParams& p, uint8_t* mem, const Four& here, const float (&x)[16]) {
        const int lane = threadIdx.x & 31, unit = lane & 3, column = lane & 15;
        uint32_t there = 0;                                       // bit r: row r of the warp is one
#pragma unroll
        for (int i = 0; i < 4; i++) {
            *reinterpret_cast<float4*>(mem + (8 * i + (lane >> 2)) * 64 + ((unit ^ (((8 * i + (lane >> 2)) >> 1) & 3)) << 4)) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            const uint32_t four = __ballot_sync(0xffffffffu, rows >> i & 1);      // (a row's four lanes say the same)
#pragma unroll
            for (int r = 0; r < 8; r++) there |= (four >> (4 * r) & 1u) << (8 * i + r);
        }
        __syncwarp();
        const bool inside = column < here.left + 4 * unit;
        TOut* to = static_cast<TOut*>(p.out) + here.at - (lane >> 2) * p.N - 4 * unit + (lane >> 4) * p.N + column;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int row = 2 * i + (lane >> 4);
            const float v = *reinterpret_cast<const float*>(mem + row * 64 + (((column >> 2) ^ ((row >> 1) & 3)) << 4) + (column & 3) * 4);
            if (inside && (there >> row & 1)) to[0] = ib::from_f32<TOut>(v);
            to += 2 * p.N;
        }
        __syncwarp();
    }
};

}  // namespace act
}  // namespace ib
