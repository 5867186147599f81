// Beam search's selection (elb_beam_select_dev): of the candidates (row b, token t) of a group, scored
// d_scores[b] + (x_bt - log sum_u exp x_bu) in double precision, the k best.
//
// Bound by memory: the logits are read once. A row is cut into chunks over many blocks; a block leaves its chunk's maximum,
// its sum of exponentials behind that maximum and the chunk's k best logits. The block of a group that arrives last... is a
// second launch: one block per group joins its rows' sums in chunk order and merges the candidates.
#include <algorithm>
#include <cmath>

#include "kv.cuh"

namespace elb {

namespace {

constexpr int BS_THREADS = 256, BS_WARPS = 8, BS_PER = 16, BS_CHUNK = BS_THREADS * BS_PER, BS_MAXK = 64;

struct BeamChunk { double sum; float mx; int pad; };

// order of a logit as an unsigned number; 0: not a candidate (-infinity or NaN)
__device__ __forceinline__ unsigned beam_key(float x) {
    const unsigned u = __float_as_uint(x);
    return x > -INFINITY ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ float beam_logit(unsigned key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// larger logit first, then the lower token
__device__ __forceinline__ unsigned long long beam_pack(unsigned key, int token) {
    return key ? (static_cast<unsigned long long>(key) << 32) | unsigned(~token) : 0ull;
}
__device__ __forceinline__ unsigned long long warp_best(unsigned long long v) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, unsigned(v >> 32));
    const unsigned lo = __reduce_max_sync(0xffffffffu, unsigned(v >> 32) == hi ? unsigned(v) : 0u);
    return (static_cast<unsigned long long>(hi) << 32) | lo;
}

__global__ void __launch_bounds__(BS_THREADS) k_beam_chunks(const float* __restrict__ logits, int64_t ld, int n, int k,
                                                            const uint32_t* __restrict__ allowed, int64_t allowed_ld,
                                                            BeamChunk* __restrict__ parts, unsigned long long* __restrict__ cand) {
    __shared__ unsigned long long lists[BS_WARPS * BS_MAXK];
    __shared__ float red_f[BS_WARPS];
    __shared__ double red_d[BS_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, chunks = gridDim.x;
    const int64_t row = blockIdx.y, slot = row * chunks + blockIdx.x;
    const float* x = logits + row * ld;
    const uint32_t* mask = allowed ? allowed + row * allowed_ld : nullptr;
    const int base = int(blockIdx.x) * BS_CHUNK + tid;
    float v[BS_PER], mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < BS_PER; ++j) {
        const int i = base + j * BS_THREADS;
        v[j] = i < n ? __ldcg(x + i) : -INFINITY;
        mx = fmaxf(mx, v[j]);
    }
    mx = warp_max(mx);
    if (lane == 0) red_f[warp] = mx;
    __syncthreads();
    for (int w = 0; w < BS_WARPS; ++w) mx = fmaxf(mx, red_f[w]);
    const double from = mx == -INFINITY ? 0.0 : double(mx);
    double sum = 0.0;
#pragma unroll 1
    for (int j = 0; j < BS_PER; ++j) {
        const int i = base + j * BS_THREADS;
        if (i < n) sum += exp(double(__ldcg(x + i)) - from);
    }
    sum = warp_sum(sum);
    if (lane == 0) red_d[warp] = sum;
    unsigned long long key[BS_PER];
#pragma unroll
    for (int j = 0; j < BS_PER; ++j) {
        const int i = base + j * BS_THREADS;
        key[j] = i < n && (!mask || ((mask[i >> 5] >> (i & 31)) & 1u)) ? beam_pack(beam_key(v[j]), i) : 0ull;
    }
    for (int r = 0; r < k; ++r) {
        unsigned long long best = key[0];
#pragma unroll
        for (int j = 1; j < BS_PER; ++j) best = key[j] > best ? key[j] : best;
        best = warp_best(best);
        if (lane == 0) lists[warp * k + r] = best;
#pragma unroll
        for (int j = 0; j < BS_PER; ++j)
            if (key[j] == best) key[j] = 0ull;
    }
    __syncthreads();
    if (warp) return;
    int at = 0;
    for (int r = 0; r < k; ++r) {
        const unsigned long long head = lane < BS_WARPS && at < k ? lists[lane * k + at] : 0ull;
        const unsigned long long best = warp_best(head);
        if (best && head == best) ++at;
        if (lane == 0) cand[slot * k + r] = best;
    }
    if (lane == 0) {
        double t = 0.0;
        for (int w = 0; w < BS_WARPS; ++w) t += red_d[w];
        parts[slot].sum = t;
        parts[slot].mx = mx;
    }
}

// One block per group, a warp per row in turn: the row's log-sum-exp and its k best in order; then one warp merges the rows.
__global__ void __launch_bounds__(BS_THREADS) k_beam_join(const BeamChunk* __restrict__ parts, const unsigned long long* __restrict__ cand,
                                                          int chunks, int beams, int k, const double* __restrict__ scores,
                                                          int* __restrict__ parent, int* __restrict__ token, double* __restrict__ score) {
    extern __shared__ unsigned long long best_of[];  // [beams][k]
    __shared__ double lse[64];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = warp; b < beams; b += BS_WARPS) {
        const int64_t row = int64_t(blockIdx.x) * beams + b;
        const BeamChunk* p = parts + row * chunks;
        float M = -INFINITY;
        for (int i = lane; i < chunks; i += 32) M = fmaxf(M, p[i].mx);
        M = warp_max(M);
        double t = 0.0;
        for (int i = lane; i < chunks; i += 32) t += p[i].sum * exp(double(p[i].mx) - double(M));
        t = warp_sum(t);
        if (lane == 0) lse[b] = double(M) + log(t);
        // a candidate that is taken is passed over by what follows it: the next best is the largest below it
        const unsigned long long* c = cand + row * chunks * k;
        unsigned long long below = ~0ull;
        for (int r = 0; r < k; ++r) {
            unsigned long long h = 0ull;
            for (int i = lane; i < chunks * k; i += 32) {
                const unsigned long long u = c[i];
                if (u < below && u > h) h = u;
            }
            below = warp_best(h);
            if (lane == 0) best_of[b * k + r] = below;
            if (!below) below = 0ull;
        }
    }
    __syncthreads();
    if (warp) return;
    int at[2] = {0, 0};  // lane holds rows lane and lane + 32
    for (int r = 0; r < k; ++r) {
        double s = -INFINITY;
        int b = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = lane + 32 * j;
            if (i >= beams || at[j] >= k) continue;
            const unsigned long long u = best_of[i * k + at[j]];
            const double x = u ? scores[int64_t(blockIdx.x) * beams + i] + (double(beam_logit(unsigned(u >> 32))) - lse[i]) : -INFINITY;
            if (x > s && x < INFINITY) { s = x; b = i; }
        }
        for (int o = 16; o > 0; o >>= 1) {
            const double s2 = __shfl_xor_sync(0xffffffffu, s, o);
            const int b2 = __shfl_xor_sync(0xffffffffu, b, o);
            if (s2 > s || (s2 == s && b2 < b)) { s = s2; b = b2; }
        }
        const bool some = b < beams;
        if (lane == 0) {
            const int64_t w = int64_t(blockIdx.x) * k + r;
            score[w] = some ? s : -INFINITY;
            parent[w] = some ? int(blockIdx.x) * beams + b : -1;
        }
        if (some && lane == (b & 31)) {
            const int j = b >> 5;
            token[int64_t(blockIdx.x) * k + r] = int(~unsigned(best_of[b * k + at[j]]));
            ++at[j];
        } else if (!some && lane == 0) {
            token[int64_t(blockIdx.x) * k + r] = -1;
        }
    }
}

size_t chunks_of(int n) { return size_t(n + BS_CHUNK - 1) / BS_CHUNK; }

}  // namespace

size_t beam_select_work(int n_vocab, int n_group, int beams, int k) {
    if (n_vocab <= 0 || n_group < 0 || beams <= 0 || beams > 64 || k <= 0 || k > BS_MAXK || int64_t(n_group) * beams > 65535) return 0;
    return std::max<size_t>(256, size_t(n_group) * beams * chunks_of(n_vocab) * (sizeof(BeamChunk) + size_t(k) * 8));
}

int beam_select_launch(int device, const float* logits, int64_t ld, int n_vocab, int n_group, int beams, const double* scores,
                       const uint32_t* allowed, int64_t allowed_ld, int k, int* parent, int* token, double* score, void* work, size_t work_bytes,
                       cudaStream_t s) {
    if (n_vocab <= 0 || n_group < 0 || beams <= 0 || beams > 64) return fail(ELB_ERR_INVALID, "beam_select: 1 to 64 beams and a vocabulary are needed");
    if (k < 1 || k > BS_MAXK || k > int64_t(beams) * n_vocab) return fail(ELB_ERR_INVALID, "beam_select: k must be between 1 and 64 (and at most beams * n_vocab)");
    if (n_vocab > (1 << 30) || int64_t(n_group) * beams > 65535) return fail(ELB_ERR_UNSUPPORTED, "beam_select: at most 65535 rows and 2^30 tokens");
    if (n_group == 0) return ELB_OK;
    if (!logits || !scores || !parent || !token || !score) return fail(ELB_ERR_INVALID, "beam_select: null argument");
    if (ld < n_vocab) return fail(ELB_ERR_INVALID, "beam_select: the row stride is shorter than a row");
    if (allowed && allowed_ld != 0 && allowed_ld < (int64_t(n_vocab) + 31) / 32) return fail(ELB_ERR_INVALID, "beam_select: the mask's row stride is shorter than a row");
    if (!work || work_bytes < beam_select_work(n_vocab, n_group, beams, k)) return fail(ELB_ERR_INVALID, "beam_select: the work buffer is too small");
    if (reinterpret_cast<uintptr_t>(work) % 256) return fail(ELB_ERR_INVALID, "beam_select: the work buffer must start on a 256-byte boundary");
    DeviceScope on(device);
    if (on.rc != ELB_OK) return on.rc;
    const int rows = n_group * beams, chunks = int(chunks_of(n_vocab));
    auto* parts = static_cast<BeamChunk*>(work);
    auto* cand = reinterpret_cast<unsigned long long*>(parts + size_t(rows) * chunks);
    k_beam_chunks<<<dim3(unsigned(chunks), unsigned(rows)), BS_THREADS, 0, s>>>(logits, ld, n_vocab, k, allowed, allowed_ld, parts, cand);
    ELB_CUDA(cudaGetLastError());
    k_beam_join<<<unsigned(n_group), BS_THREADS, size_t(beams) * k * 8, s>>>(parts, cand, chunks, beams, k, scores, parent, token, score);
    ELB_CUDA(cudaGetLastError());
    return ELB_OK;
}

}  // namespace elb
