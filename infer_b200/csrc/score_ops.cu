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
// A row is shared by the CTAs of a cluster, each taking a contiguous slice of its 16-byte units (up to three elements before the first and behind
// the last whole unit are the first CTA's beside them). A thread takes every THREADS-th unit, four at a time, and the next four are
// requested before these are looked at; the statistics need no barrier until the end.
// The alternatives cost the stream one comparison for four units (the thread's largest element and its id): the `top` best of all elements
// lie with at most `top` threads, those whose largest reaches the top-th largest of the threads'.  A bound on that is enough: the top-th
// of the largest of 64 groups of 8 threads.  The elements of the few threads that reach it are read again (from L2), those that
// reach the bound themselves go into shared memory beside the list of what came before, and every entry counts the entries that beat it.
// A slice goes in segments, so that the room in shared memory is enough whatever the row holds: where the bound lets through more
// threads than fit, the threads' own keys are compared and exactly `top` remain. (With a list that each chunk's elements were compared with,
// 64 rows took 43 us instead of 16.5; bound checks of the row's ends at every unit were another third.)
// Bound by HBM for many rows (1,024 x 152,064 99.5 us, 6.2 TB/s), for few by its steps one after the other: one row of 151,936 in a cluster of eight
// 4.8 us without alternatives, 8.0 with five, of which the stream takes 2.7, what finds the five 1.9, the join 2.5.
constexpr int THREADS = 512, UNITS = 4, GROUPS = THREADS / 8;
constexpr int SEGMENT = 48;                                              // units of a thread in a segment
constexpr int MAX_TOP = ib::score::MAX_TOP;
constexpr int ROOM = 5120;                                               // keys of a segment's candidates
static_assert(ROOM >= MAX_TOP * SEGMENT * 4 + 6 + 8 * MAX_TOP && SEGMENT % UNITS == 0 && MAX_TOP <= GROUPS, "the candidates fit");

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

// Entries i of keys[0, n) that fewer than `top` others beat, called with (how many beat it, the key) by one thread each. Unequal keys, 0: none.
template <typename F> __device__ __forceinline__ void ranked(const unsigned long long* keys, int n, int top, F&& put) {
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const unsigned long long k = keys[i];
        int above = 0, j = 0;
        for (; j + 4 <= n; j += 4) {
            const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(keys + j), b = *reinterpret_cast<const ulonglong2*>(keys + j + 2);
            above += (a.x > k) + (a.y > k) + (b.x > k) + (b.y > k);
        }
        for (; j < n; j++) above += keys[j] > k;
        if (k != 0 && above < top) put(above, k);
    }
}

template <int CL, bool TOP>
__global__ void __launch_bounds__(THREADS, 2)
token_logprobs_kernel(const Params p) {
    extern __shared__ __align__(16) unsigned long long keys[];           // TOP: the list [MAX_TOP], candidates [ROOM], the new list [MAX_TOP]
    __shared__ Stats red[THREADS / 32];
    __shared__ float red_m[THREADS / 32];
    __shared__ Stats parts[CL];                                           // of the cluster's CTAs, in the first
    __shared__ __align__(16) unsigned long long lists[TOP ? CL * MAX_TOP : 1];
    __shared__ unsigned long long best[TOP ? GROUPS : 1], bound;
    __shared__ int n_keys;
    const int rank = CL > 1 ? int(cg::this_cluster().block_rank()) : 0;
    const int64_t b = blockIdx.x / CL;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* row = p.logits + b * p.vocab;
    // whole units start `lead` elements into the row
    const int lead = int(min(int64_t((4 - ((reinterpret_cast<uintptr_t>(row) >> 2) & 3)) & 3), p.vocab));
    const int64_t n_units = (p.vocab - lead) / 4;
    const int edges = lead + int((p.vocab - lead) & 3);                   // elements outside of whole units
    const int64_t per = (n_units + CL - 1) / CL, u_lo = min(n_units, per * rank);
    const int mine = int(min(n_units, u_lo + per) - u_lo);                // units of this CTA
    const float4* units = reinterpret_cast<const float4*>(row + lead) + u_lo;
    const uint32_t id0 = uint32_t(lead + 4 * u_lo);                       // of this CTA's first unit's first element
    unsigned long long* found = keys + MAX_TOP;
    if (TOP) {
        if (threadIdx.x < MAX_TOP) keys[threadIdx.x] = keys[MAX_TOP + ROOM + threadIdx.x] = 0;
        if (threadIdx.x == 0) { n_keys = 0; bound = 0; }
        __syncthreads();
    }
    if (CL > 1) cg::this_cluster().barrier_arrive();                      // (waited for before another CTA's shared memory is written)
    ib::pdl_wait();
    int token = -1;
    float at = 0.0f;
    if (rank == 0 && threadIdx.x == 0 && p.tokens) {
        token = p.tokens[b];
        if (token >= 0 && token < p.vocab) at = row[token];
    }
    auto fetch = [&](int i) { return i < mine ? units[i] : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); };
    Stats st;
    st.clear();
    float4 next[UNITS];
#pragma unroll
    for (int j = 0; j < UNITS; j++) next[j] = fetch(j * THREADS + int(threadIdx.x));
    if (rank == 0 && int(threadIdx.x) < edges) {
        const int64_t e = int(threadIdx.x) < lead ? int64_t(threadIdx.x) : p.vocab - edges + threadIdx.x;
        float z[1] = {row[e]};
        if (TOP && z[0] > -INFINITY) found[atomicAdd(&n_keys, 1)] = ib::score::key(z[0], uint32_t(e));
        if (p.cap > 0.0f) {
            float l[1];
            ib::score::cap_logits<1>(l, z, p.scale, p.cap);
            st.add<1>(l, l[0]);
        } else {
            st.add<1>(z, z[0], p.scale);
        }
    }
    int s0 = 0;
    do {
        const int s1 = min(mine, s0 + SEGMENT * THREADS);
        float largest = -INFINITY;
        int largest_at = 0;                                               // element of this CTA's units
        for (int i0 = s0; i0 < s1; i0 += UNITS * THREADS) {
            float z[UNITS * 4];
#pragma unroll
            for (int j = 0; j < UNITS; j++) { z[4 * j] = next[j].x; z[4 * j + 1] = next[j].y; z[4 * j + 2] = next[j].z; z[4 * j + 3] = next[j].w; }
#pragma unroll
            for (int j = 0; j < UNITS; j++) next[j] = fetch(i0 + (UNITS + j) * THREADS + int(threadIdx.x));
            const float m = ib::score::largest_of<UNITS * 4>(z);
            if (TOP && m > largest) {
                largest = m;
                int which = 0;
#pragma unroll
                for (int i = UNITS * 4 - 1; i >= 0; i--) which = z[i] == m ? i : which;
                largest_at = 4 * (i0 + (which >> 2) * THREADS + int(threadIdx.x)) + (which & 3);
            }
            if (p.cap > 0.0f) {
                float l[UNITS * 4];
                ib::score::cap_logits<UNITS * 4>(l, z, p.scale, p.cap);
                st.add<UNITS * 4>(l, ib::score::largest_of<UNITS * 4>(l));
            } else {
                st.add<UNITS * 4>(z, m, p.scale);
            }
        }
        s0 += SEGMENT * THREADS;
        if (TOP) {
            const unsigned long long last = keys[p.top - 1];              // 0: fewer than top so far
            const unsigned long long mine_best = largest > -INFINITY ? ib::score::key(largest, id0 + largest_at) : 0;
            bool in = mine_best > last;
            const int any = __syncthreads_count(in), held = n_keys;        // held: elements outside of whole units
            if (any + held == 0) continue;
            unsigned long long g = mine_best;
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, g, o);
                g = other > g ? other : g;
            }
            if ((lane & 7) == 0) best[threadIdx.x >> 3] = g;
            __syncthreads();
            const unsigned long long g0 = best[lane], g1 = best[lane + 32];
#pragma unroll
            for (int i = 0; i < GROUPS / (THREADS / 32); i++) {           // a warp looks where a few of the groups stand among all
                const unsigned long long k = best[warp * (GROUPS / (THREADS / 32)) + i];
                const int above = __popc(__ballot_sync(0xffffffffu, g0 > k)) + __popc(__ballot_sync(0xffffffffu, g1 > k));
                if (lane == 0 && k != 0 && above == p.top - 1) bound = k;
            }
            __syncthreads();
            unsigned long long least = max(bound, last + 1);
            in = mine_best >= least;
            const int begin = s0 - SEGMENT * THREADS, reach = (s1 - begin + THREADS - 1) / THREADS;        // units of a thread
            if (__syncthreads_count(in) * reach * 4 + held > ROOM) {
                if (in) found[6 + atomicAdd(&n_keys, 1) - held] = mine_best;
                __syncthreads();
                ranked(found + 6, n_keys - held, p.top, [&](int above, unsigned long long k) { if (above == p.top - 1) bound = k; });
                __syncthreads();
                least = max(bound, last + 1);
                in = mine_best >= least;
                if (threadIdx.x == 0) n_keys = held;
                __syncthreads();
            }
            // a warp reads its chosen threads' units again, a thread at a time
            for (uint32_t todo = __ballot_sync(0xffffffffu, in); todo; todo &= todo - 1) {
                const int t = warp * 32 + __ffs(todo) - 1;
                for (int j = lane; j < reach; j += 32) {
                    const int i = begin + j * THREADS + t;
                    if (i >= s1) break;
                    const float4 f = units[i];
                    const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const unsigned long long key = v[k] > -INFINITY ? ib::score::key(v[k], id0 + 4 * i + k) : 0;
                        if (key >= least) found[atomicAdd(&n_keys, 1)] = key;
                    }
                }
            }
            __syncthreads();
            ranked(keys, MAX_TOP + n_keys, p.top, [&](int above, unsigned long long k) { keys[MAX_TOP + ROOM + above] = k; });
            __syncthreads();
            if (threadIdx.x < MAX_TOP) {
                keys[threadIdx.x] = keys[MAX_TOP + ROOM + threadIdx.x];
                keys[MAX_TOP + ROOM + threadIdx.x] = 0;
            }
            if (threadIdx.x == 0) { n_keys = 0; bound = 0; }
            __syncthreads();
        }
    } while (s0 < mine);
    ib::pdl_launch_dependents();
    // the block's maximum, each thread rescaled to it once, sums
    const float warp_m = ib::warp_max(st.m);
    if (lane == 0) red_m[warp] = warp_m;
    __syncthreads();
    st.raise(ib::warp_max(red_m[lane & (THREADS / 32 - 1)]));
    st.s = ib::warp_sum(st.s);
    st.d = ib::warp_sum(st.d);
    if (lane == 0) red[warp] = st;
    __syncthreads();
    if (warp == 0) {
        st.s = ib::warp_sum(lane < THREADS / 32 ? red[lane].s : 0.0f);
        st.d = ib::warp_sum(lane < THREADS / 32 ? red[lane].d : 0.0f);
    }
    if (CL > 1) {
        auto cluster = cg::this_cluster();
        cluster.barrier_wait();
        if (threadIdx.x == 0) *cluster.map_shared_rank(&parts[rank], 0) = st;
        if (TOP && threadIdx.x < p.top) *cluster.map_shared_rank(&lists[rank * p.top + threadIdx.x], 0) = keys[threadIdx.x];
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
        ib::score::finish(st, token, at, p.scale, p.cap, p.vocab, p.logprob + b, p.entropy + b, p.status);
    }
    if (TOP) {
        __syncthreads();
        st = red[0];
        bool any = false;
        ranked(CL > 1 ? lists : keys, CL > 1 ? CL * p.top : MAX_TOP, p.top, [&](int above, unsigned long long k) {
            any = true;
            p.top_ids[b * p.top + above] = int(ib::score::key_id(k));
            p.top_logprobs[b * p.top + above] = ib::score::logprob_of(st, ib::score::key_value(k), p.scale, p.cap);
        });
        const int filled = __syncthreads_count(any);                      // (CL x MAX_TOP entries: a thread has one at most)
        if (threadIdx.x >= filled && threadIdx.x < p.top) {
            p.top_ids[b * p.top + threadIdx.x] = -1;
            p.top_logprobs[b * p.top + threadIdx.x] = -INFINITY;
        }
    }
}

template <int CL, bool TOP>
int launch_logprobs(const Params& p, int64_t rows, cudaStream_t stream) {
    const size_t smem = TOP ? size_t(ROOM + 2 * MAX_TOP) * 8 : 0;
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
    if (vocab <= 0 || vocab >= (1LL << 30)) return ib::fail(IB_ERR_ARG, "token_logprobs: vocabulary %lld out of range", (long long)vocab);
    if (rows > 0x7fffffff / 8) return ib::fail(IB_ERR_ARG, "token_logprobs: too many rows (%lld)", (long long)rows);
    if (top < 0 || top > MAX_TOP) return ib::fail(IB_ERR_ARG, "token_logprobs: 0 to %d alternatives, not %d", MAX_TOP, top);
    if (!logprob || !entropy || (top && (!top_ids || !top_logprobs))) return ib::fail(IB_ERR_ARG, "token_logprobs: results are needed");
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
