// How likely the answers of a model are: log probabilities of given tokens, entropies and the likeliest alternatives, from rows of float
// logits; and the last step of a product with an activation, for the sizes that no product kernel finishes by itself.
//
// A row of logits l (of z: l = scale z, or with a cap l = cap tanh(scale z / cap)): with m = max l, S = sum exp(l - m) and
// D = sum exp(l - m) (l - m),  logprob(t) = (l[t] - m) - ln S,  entropy = ln S - D / S.  One pass: every thread keeps its own m, S and D, and
// where its maximum rises by x, D becomes e^-x (D - x S) and S becomes e^-x S.  An element of -inf adds nothing (0 * -inf is left out of D);
// a row without any other has log probability -inf and entropy 0; a NaN or +inf makes both NaN.
#include "common.cuh"
#include "score.cuh"

#include <cooperative_groups.h>

IB_DEFINE_LAST_ERROR()

namespace {

namespace cg = cooperative_groups;
using ib::score::Stats;
using bf16 = __nv_bfloat16;

// ------------------------------------------------------------------------------------------------ from logits
// A row is shared by the CTAs of a cluster, each taking a contiguous slice in chunks of THREADS x 16 elements; a thread holds four
// 16-byte units of a chunk, and the next chunk's are requested before this one is looked at.  The statistics need no barrier until
// the end.  For the alternatives a CTA keeps the best `top` keys of what it has seen, sorted, in shared memory; a chunk in which no element
// beats the last of them costs one barrier.  Otherwise what beats it is appended behind the list, every entry counts the entries that
// beat it, and those beaten by fewer than `top` are the new list.  In a first chunk nearly everything would be appended, so there a
// lower bound comes first: of the 32 half-warps' best keys the top-th; only `top` half-warps hold keys that reach it, so that
// MAX_TOP x 256 places are enough whatever the row holds.
constexpr int THREADS = 512, UNITS = 4;
constexpr int MAX_TOP = ib::score::MAX_TOP, GROUPS = THREADS / 16;
constexpr int ROOM = MAX_TOP + MAX_TOP * 16 * 4 * UNITS;                 // the list, and what one chunk may append
static_assert(GROUPS == 32, "a warp compares the half-warps' best keys");

struct Params {
    const float* logits;
    int64_t vocab;
    const int* tokens;           // or null
    int top;
    float scale, cap;
    float* logprob;
    float* entropy;
    int* top_ids;
    float* top_logprobs;
    int* status;                 // or null
};

template <int CL, bool TOP>
__global__ void __launch_bounds__(THREADS, 2)
token_logprobs_kernel(const Params p) {
    extern __shared__ __align__(16) unsigned long long keys[];           // TOP: [ROOM], then the new list [MAX_TOP]
    __shared__ Stats red[THREADS / 32];
    __shared__ Stats parts[CL];                                           // of the cluster's CTAs, in the first
    __shared__ unsigned long long lists[TOP ? CL * MAX_TOP : 1];
    __shared__ unsigned long long best[GROUPS];
    __shared__ int n_keys;
    const int rank = CL > 1 ? int(cg::this_cluster().block_rank()) : 0;
    const int64_t b = blockIdx.x / CL;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* row = p.logits + b * p.vocab;
    // the row's first element sits `ahead` floats behind a 16-byte boundary: units are counted from that boundary
    const int ahead = int((reinterpret_cast<uintptr_t>(row) >> 2) & 3);
    const int64_t n_units = (p.vocab + ahead + 3) / 4;
    const int64_t per = ((n_units + CL - 1) / CL + 31) / 32 * 32, u_lo = min(n_units, per * rank), u_hi = min(n_units, u_lo + per);
    const int n_chunks = int((u_hi - u_lo + THREADS * UNITS - 1) / (THREADS * UNITS));
    if (TOP) {
        if (threadIdx.x < MAX_TOP) keys[threadIdx.x] = keys[ROOM + threadIdx.x] = 0;
        if (threadIdx.x == 0) n_keys = 0;
        __syncthreads();
    }
    if (CL > 1) cg::this_cluster().barrier_arrive();                      // (waited for before another CTA's shared memory is written)
    ib::pdl_wait();
    const bool asked = rank == 0 && threadIdx.x == 0;
    int token = -1;
    float at = 0.0f;
    if (asked && p.tokens) {
        token = p.tokens[b];
        if (token >= 0 && token < p.vocab) at = row[token];
    }
    auto fetch = [&](int chunk, float (&v)[UNITS * 4]) {
#pragma unroll
        for (int j = 0; j < UNITS; j++) {
            const int64_t u = u_lo + int64_t(chunk) * (THREADS * UNITS) + j * THREADS + threadIdx.x, e = 4 * u - ahead;
            if (u < u_hi && e >= 0 && e + 4 <= p.vocab) {
                const float4 f = __ldcs(reinterpret_cast<const float4*>(row + e));
                v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) v[4 * j + k] = u < u_hi && e + k >= 0 && e + k < p.vocab ? row[e + k] : -INFINITY;
            }
        }
    };
    Stats st;
    st.clear();
    float next[UNITS * 4];
    if (n_chunks > 0) fetch(0, next);
    for (int chunk = 0; chunk < n_chunks; chunk++) {
        float z[UNITS * 4];
#pragma unroll
        for (int i = 0; i < UNITS * 4; i++) z[i] = next[i];
        if (chunk + 1 < n_chunks) fetch(chunk + 1, next);
        if (TOP) {
            // (keys are made where they are needed: 64-bit comparisons of 16 elements would cost more than the statistics)
            const int64_t e0 = 4 * (u_lo + int64_t(chunk) * (THREADS * UNITS) + threadIdx.x) - ahead;
            auto key_of = [&](int i) { return ib::score::key(z[i], uint32_t(e0 + int64_t(i / 4) * (THREADS * 4) + (i & 3))); };
            const unsigned long long last = keys[p.top - 1];              // 0: fewer than top so far
            const float floor = last ? ib::score::key_value(last) : -INFINITY;
            bool any = false;
#pragma unroll
            for (int i = 0; i < UNITS * 4; i++) any |= z[i] > floor;         // (an equal one has a higher id than what is in the list)
            const int busy = __syncthreads_count(any);
            if (busy) {
                unsigned long long bound = last + 1;
                if (busy * (UNITS * 4) > ROOM - MAX_TOP) {
                    unsigned long long mine = 0;
#pragma unroll
                    for (int i = 0; i < UNITS * 4; i++)
                        if (z[i] > -INFINITY) { const unsigned long long k = key_of(i); mine = k > mine ? k : mine; }
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1) {
                        const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, o);
                        mine = other > mine ? other : mine;
                    }
                    if ((lane & 15) == 0) best[threadIdx.x >> 4] = mine;
                    __syncthreads();
                    const unsigned long long g = best[lane];
                    int beaten = 0;
#pragma unroll
                    for (int o = 0; o < 32; o++) { const unsigned long long other = __shfl_sync(0xffffffffu, g, o); beaten += other > g || (other == g && o < lane); }
                    const unsigned int who = __ballot_sync(0xffffffffu, beaten == p.top - 1);
                    const unsigned long long kth = __shfl_sync(0xffffffffu, g, __ffs(who) - 1);
                    bound = kth > bound ? kth : bound;
                }
                if (any) {
#pragma unroll
                    for (int i = 0; i < UNITS * 4; i++) {
                        if (!(z[i] > -INFINITY)) continue;
                        const unsigned long long k = key_of(i);
                        if (k >= bound) keys[MAX_TOP + atomicAdd(&n_keys, 1)] = k;
                    }
                }
                __syncthreads();
                const int n = MAX_TOP + n_keys;
                for (int i = threadIdx.x; i < n; i += THREADS) {
                    const unsigned long long k = keys[i];
                    if (k == 0) continue;
                    int above = 0;
                    for (int j = 0; j < n; j++) above += keys[j] > k;
                    if (above < p.top) keys[ROOM + above] = k;
                }
                __syncthreads();
                if (threadIdx.x < p.top) keys[threadIdx.x] = keys[ROOM + threadIdx.x];
                if (threadIdx.x == 0) n_keys = 0;
                __syncthreads();
                if (threadIdx.x < MAX_TOP) keys[ROOM + threadIdx.x] = 0;
                // (read again only behind the next chunk's barrier)
            }
        }
        if (p.cap > 0.0f) {
#pragma unroll
            for (int i = 0; i < UNITS * 4; i++) z[i] = ib::score::logit(z[i], p.scale, p.cap);
        } else if (p.scale != 1.0f) {
#pragma unroll
            for (int i = 0; i < UNITS * 4; i++) z[i] *= p.scale;
        }
        st.add<UNITS * 4>(z);
    }
    ib::pdl_launch_dependents();
    st = ib::score::warp_join(st);
    if (lane == 0) red[warp] = st;
    __syncthreads();
    if (warp == 0) {
        st.clear();
        if (lane < THREADS / 32) st = red[lane];
        st = ib::score::warp_join(st);
    }
    if (CL > 1) {
        auto cluster = cg::this_cluster();
        cluster.barrier_wait();
        if (threadIdx.x == 0) *cluster.map_shared_rank(&parts[rank], 0) = st;
        if (TOP) for (int i = threadIdx.x; i < MAX_TOP; i += THREADS) *cluster.map_shared_rank(&lists[rank * MAX_TOP + i], 0) = i < p.top ? keys[i] : 0;
        cluster.sync();
        if (rank != 0) return;
        if (warp == 0) {
            st.clear();
            if (lane < CL) st = parts[lane];
            st = ib::score::warp_join(st);
        }
    }
    if (threadIdx.x == 0) {
        red[0] = st;
        ib::score::finish(st, token, ib::score::logit(at, p.scale, p.cap), p.vocab, p.logprob ? p.logprob + b : nullptr, p.entropy ? p.entropy + b : nullptr, p.status);
    }
    if (TOP) {
        __syncthreads();
        st = red[0];
        const unsigned long long* all = CL > 1 ? lists : keys;
        const int n = CL > 1 ? CL * MAX_TOP : MAX_TOP;
        int found = 0;
        if (threadIdx.x < n) {
            const unsigned long long k = all[threadIdx.x];
            int above = 0;
            for (int j = 0; j < n; j++) above += all[j] > k;
            found = k != 0 && above < p.top;
            if (found) {
                p.top_ids[b * p.top + above] = int(ib::score::key_id(k));
                p.top_logprobs[b * p.top + above] = st.logprob(ib::score::logit(ib::score::key_value(k), p.scale, p.cap));
            }
        }
        const int filled = __syncthreads_count(found);
        if (threadIdx.x >= filled && threadIdx.x < p.top) {
            p.top_ids[b * p.top + threadIdx.x] = -1;
            p.top_logprobs[b * p.top + threadIdx.x] = -INFINITY;
        }
    }
}

template <int CL, bool TOP>
int launch_logprobs(const Params& p, int64_t rows, cudaStream_t stream) {
    const size_t smem = TOP ? size_t(ROOM + MAX_TOP) * 8 : 0;
    static ib::PerDevice allowed;
    if (const int rc = ib::allow_smem(allowed, "token_logprobs", token_logprobs_kernel<CL, TOP>, smem)) return rc;
    return ib::launch("token_logprobs", token_logprobs_kernel<CL, TOP>, dim3(unsigned(rows * CL)), dim3(THREADS), smem, stream, CL, p);
}

// ------------------------------------------------------------------------------------------------ activation and residual
// out = residual + act(z), z float [n] (a product with its bias): bound by the bytes of z, residual and out.
template <typename TOut>
__global__ void act_residual_kernel(const float* __restrict__ z, const float* residual, TOut* out, int64_t n, int act) {
    ib::pdl_wait();
    const int64_t stride = int64_t(gridDim.x) * blockDim.x;
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += stride) {
        float v = ib::score::activate(z[i], act);
        if (residual) v += residual[i];
        out[i] = ib::from_f32<TOut>(v);
    }
}

}  // namespace

IB_EXPORT int ib_max_top_logprobs() { return MAX_TOP; }

// logits float [rows, vocab]; tokens int [rows] or null; top 0 .. MAX_TOP. logprob, entropy [rows]; top_ids, top_logprobs [rows, top].
// cluster: CTAs to a row (1, 2, 4 or 8).
IB_EXPORT int ib_token_logprobs(const float* logits, int64_t rows, int64_t vocab, const int* tokens, int top, float scale, float cap, float* logprob,
                                float* entropy, int* top_ids, float* top_logprobs, int cluster, int* status, cudaStream_t stream) {
    if (rows <= 0) return IB_OK;
    if (vocab <= 0 || vocab >= 0x7fffffff) return ib::fail(IB_ERR_ARG, "token_logprobs: vocabulary %lld out of range", (long long)vocab);
    if (rows > 0x7fffffff / 8) return ib::fail(IB_ERR_ARG, "token_logprobs: too many rows (%lld)", (long long)rows);
    if (top < 0 || top > MAX_TOP) return ib::fail(IB_ERR_ARG, "token_logprobs: 0 to %d alternatives, not %d", MAX_TOP, top);
    if (!(scale > 0.0f) || !(cap >= 0.0f)) return ib::fail(IB_ERR_ARG, "token_logprobs: the scale must be positive, the cap not negative");
    const Params p{logits, vocab, tokens, top, scale, cap, logprob, entropy, top_ids, top_logprobs, status};
    switch (cluster) {
        case 1: return top ? launch_logprobs<1, true>(p, rows, stream) : launch_logprobs<1, false>(p, rows, stream);
        case 2: return top ? launch_logprobs<2, true>(p, rows, stream) : launch_logprobs<2, false>(p, rows, stream);
        case 4: return top ? launch_logprobs<4, true>(p, rows, stream) : launch_logprobs<4, false>(p, rows, stream);
        case 8: return top ? launch_logprobs<8, true>(p, rows, stream) : launch_logprobs<8, false>(p, rows, stream);
    }
    return ib::fail(IB_ERR_ARG, "token_logprobs: 1, 2, 4 or 8 CTAs to a row, not %d", cluster);
}

IB_EXPORT int ib_act_residual(const float* z, const float* residual, void* out, int64_t n, int act, int out_dtype, cudaStream_t stream) {
    if (n <= 0) return IB_OK;
    if (act < 0 || act >= ib::score::ACTIVATIONS) return ib::fail(IB_ERR_ARG, "act_residual: unknown activation %d", act);
    const int64_t blocks = (n + 1023) / 1024;
    const dim3 grid{unsigned(blocks < 148 * 16 ? blocks : 148 * 16)};
    if (out_dtype == IB_F32) return ib::launch("act_residual", act_residual_kernel<float>, grid, dim3(256), 0, stream, 1u, z, residual, (float*)out, n, act);
    if (out_dtype == IB_BF16) return ib::launch("act_residual", act_residual_kernel<bf16>, grid, dim3(256), 0, stream, 1u, z, residual, (bf16*)out, n, act);
    return ib::fail(IB_ERR_ARG, "act_residual: unknown output dtype %d", out_dtype);
}
