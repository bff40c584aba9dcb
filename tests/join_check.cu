// The kernel of score_head.cu that joins a row's chunks, by itself (test_join_chunks_gpu.py), on lists that the test writes. The launch is that of
// ib_head_logprobs: shared memory for the statistics and first keys of every chunk and for min(chunks, top) lists of `top` keys.
#include "score_head.cu"

IB_EXPORT int join_check(int64_t rows, int64_t vocab, int chunks, int n, int top, const float* stats, const void* lists, const float* at, float* logprob, float* entropy,
                         int* ids, float* logprobs, int* status, cudaStream_t stream) {
    const JoinParams j{rows, vocab, chunks, n, top, 1.0f, 0.0f, nullptr, reinterpret_cast<const float4*>(stats), static_cast<const unsigned long long*>(lists), at,
                       logprob, entropy, ids, logprobs, status};
    const size_t smem = size_t(chunks) * 24 + size_t(chunks < top ? chunks : top) * top * 8;
    return ib::launch("join_chunks", join_chunks_kernel, dim3(unsigned(rows)), dim3(JOIN_THREADS), smem, stream, 1u, j);
}
