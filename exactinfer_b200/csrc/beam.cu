// Beam search's selection (elb_beam_select_dev): of the candidates (row b, token t) of a group, scored
// d_scores[b] + (x_bt - log sum_u exp x_bu) in double precision, the k best.
//
// Bound by memory: the logits are read once. A row is cut into chunks of 4096 over many blocks; a block leaves its chunk's maximum,
// its sum of exponentials behind that maximum and the chunk's k best logits in order. A second launch, one block per group and
// a warp per row, joins the sums in chunk order, merges the lists, and picks over the rows.
//
// Exponentials are the work beside the loads: double precision, e^y = 2^(i/64) 2^n e^r with y = (64 n + i) ln 2 / 64 + r, |r| <=
// ln 2 / 128 and the Taylor sum of e^r to r^4 / 24 (4e-14 off at most), nine double operations a logit. The k best: of k groups
// of threads each has a largest logit; the smallest of these is a bound that at least k logits reach and, on logits that
// are spread at all, few more. Those are listed and each finds its place by counting the larger ones.
#include <algorithm>
#include <cmath>

#include "kv.cuh"

namespace elb {

namespace {

constexpr int BS_THREADS = 256, BS_WARPS = 8, BS_PER = 16, BS_CHUNK = BS_THREADS * BS_PER, BS_MAXK = 64;
constexpr int BS_LIST = 1024;  // logits of a chunk that may reach its bound before the slow way is taken
constexpr int BJ_STAGE = 512;  // candidates of a row that are merged in shared memory

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

// sum + e^y for -701 <= y <= 0; tab[i] = 2^(i/64). NaN stays NaN
__device__ __forceinline__ double add_exp(double sum, double y, const double* tab) {
    const double t = fma(y, 92.332482616893656769, 6755399441055744.0);  // 64 / ln 2; 1.5 * 2^52: the low word is the rounded integer
    const double r = fma(t - 6755399441055744.0, -0.010830424696249145, y);  // ln 2 / 64
    const int n = __double2loint(t);
    double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double s = tab[n & 63];
    return fma(__hiloint2double(__double2hiint(s) + ((n & ~63) << 14), __double2loint(s)), p, sum);
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// VEC: rows start on 16-byte boundaries
template <bool VEC>
__global__ void __launch_bounds__(BS_THREADS) k_beam_chunks(const float* __restrict__ logits, int64_t ld, int n, int k, int groups_log,
                                                            const uint32_t* __restrict__ allowed, int64_t allowed_ld,
                                                            BeamChunk* __restrict__ parts, unsigned long long* __restrict__ cand) {
    __shared__ unsigned long long list[BS_LIST];  // (the slow way: [warp][k])
    __shared__ double tab[64];
    __shared__ float red_f[BS_WARPS], red_b[BS_WARPS];
    __shared__ double red_d[BS_WARPS];
    __shared__ int count;
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, chunks = gridDim.x;
    const int64_t row = blockIdx.y, slot = row * chunks + blockIdx.x;
    const float* x = logits + row * ld;
    const uint32_t* mask = allowed ? allowed + row * allowed_ld : nullptr;
    const int base = int(blockIdx.x) * BS_CHUNK;
    auto token = [&](int j) { return base + 4 * (BS_THREADS * (j / 4) + tid) + (j & 3); };  // of a thread's j-th logit
    float v[BS_PER];
#pragma unroll
    for (int q = 0; q < BS_PER / 4; ++q) {
        const int i = token(4 * q);
        if (VEC && i + 3 < n) {
            *reinterpret_cast<float4*>(v + 4 * q) = __ldcg(reinterpret_cast<const float4*>(x + i));
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * q + c] = i + c < n ? __ldcg(x + i + c) : -INFINITY;
        }
    }
    unsigned off = 0;  // bit j: logit j may not be picked
    if (mask) {
#pragma unroll
        for (int q = 0; q < BS_PER / 4; ++q) {
            const int i = token(4 * q);
            off |= (i < n ? ~(mask[i >> 5] >> (i & 31)) & 15u : 15u) << (4 * q);
        }
    }
    if (tid < 64) tab[tid] = exp2(tid / 64.0);
    if (tid == 0) count = 0;
    float mx = -INFINITY;  // (NaN is passed over here and spoils the sum below)
#pragma unroll
    for (int j = 0; j < BS_PER; ++j) mx = fmaxf(mx, v[j]);
    float best = mx;  // the largest that may be picked
    if (mask) {
        best = -INFINITY;
#pragma unroll
        for (int j = 0; j < BS_PER; ++j) best = (off >> j) & 1u ? best : fmaxf(best, v[j]);
    }
    float bound = best;
    for (int o = 1; o < 32 >> max(0, groups_log - 3); o <<= 1) bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, o));  // of a group of threads
    for (int o = 16; o > 0; o >>= 1) bound = fminf(bound, __shfl_xor_sync(0xffffffffu, bound, o));
    mx = warp_max(mx);
    if (lane == 0) { red_f[warp] = mx; red_b[warp] = bound; }
    __syncthreads();
    bound = red_b[0];
#pragma unroll
    for (int w = 0; w < BS_WARPS; ++w) { mx = fmaxf(mx, red_f[w]); bound = fminf(bound, red_b[w]); }
    if (best >= bound && best > -INFINITY) {  // (the order of the list does not matter: places are counted)
#pragma unroll
        for (int j = 0; j < BS_PER; ++j)
            if (v[j] >= bound && v[j] > -INFINITY && !((off >> j) & 1u)) {
                const int at = atomicAdd(&count, 1);
                if (at < BS_LIST) list[at] = beam_pack(beam_key(v[j]), token(j));
            }
    }
    // Terms below e^-700 of the largest, and places behind the row's end, count as e^-700: nothing beside the largest's 1. A row
    // with +infinity has no log-sum-exp.
    double sum = mx < INFINITY ? 0.0 : double(NAN);
    if (mx != -INFINITY) {
        const float low = mx - 700.f;
        const double from = mx;
#pragma unroll
        for (int j = 0; j < BS_PER; ++j) sum = add_exp(sum, double(max_nan(v[j], low)) - from, tab);
    } else {
#pragma unroll
        for (int j = 0; j < BS_PER; ++j) sum = v[j] != v[j] ? double(NAN) : sum;
    }
    sum = warp_sum(sum);
    if (lane == 0) red_d[warp] = sum;
    __syncthreads();
    const int have = count;
    if (tid == 0) {
        double t = 0.0;
        for (int w = 0; w < BS_WARPS; ++w) t += red_d[w];
        parts[slot].sum = t;
        parts[slot].mx = mx;
    }
    if (have <= BS_LIST) {  // a candidate's place: how many are larger
        for (int c = tid; c < have; c += BS_THREADS) {
            const unsigned long long me = list[c];
            int place = 0;
            for (int o = 0; o < have; ++o) place += list[o] > me;
            if (place < k) cand[slot * k + place] = me;
        }
        for (int r = have + tid; r < k; r += BS_THREADS) cand[slot * k + r] = 0ull;
        return;
    }
    // many logits at the bound (equal ones): every warp its k best one by one, then a merge of the warps' lists
    __syncthreads();
    for (int r = 0; r < k; ++r) {
        unsigned long long most = 0ull;
#pragma unroll
        for (int j = 0; j < BS_PER; ++j) {
            const unsigned long long u = (off >> j) & 1u ? 0ull : beam_pack(beam_key(v[j]), token(j));
            most = u > most ? u : most;
        }
        most = warp_best(most);
        if (lane == 0) list[warp * k + r] = most;
#pragma unroll
        for (int j = 0; j < BS_PER; ++j)
            if (most && token(j) == int(~unsigned(most))) off |= 1u << j;
    }
    __syncthreads();
    if (warp) return;
    int at = 0;
    for (int r = 0; r < k; ++r) {
        const unsigned long long head = lane < BS_WARPS && at < k ? list[lane * k + at] : 0ull;
        const unsigned long long best = warp_best(head);
        if (best && head == best) ++at;
        if (lane == 0) cand[slot * k + r] = best;
    }
}

// One block per group, a warp per row in turn: the row's log-sum-exp and its k best in order; then one warp merges the rows.
__global__ void __launch_bounds__(BS_THREADS) k_beam_join(const BeamChunk* __restrict__ parts, const unsigned long long* __restrict__ cand,
                                                          int chunks, int beams, int k, const double* __restrict__ scores,
                                                          int* __restrict__ parent, int* __restrict__ token, double* __restrict__ score) {
    extern __shared__ unsigned long long best_of[];  // [beams][k], then [warp][BJ_STAGE]
    unsigned long long* stage = best_of + beams * k;
    pdl_wait();
    __shared__ double lse[64];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = warp; b < beams; b += BS_WARPS) {
        const int64_t row = int64_t(blockIdx.x) * beams + b;
        // merge of the chunks' lists; a lane holds chunks lane, lane + 32, ... and looks again only when one of its own was taken
        const unsigned long long* c = cand + row * chunks * k;
        if (chunks <= 64 && chunks * k <= BJ_STAGE) {
            unsigned long long* st = stage + warp * BJ_STAGE;
            for (int i = lane; i < chunks * k; i += 32) st[i] = c[i];
            c = st;
        }
        const BeamChunk* p = parts + row * chunks;
        float M = -INFINITY;
        for (int i = lane; i < chunks; i += 32) M = fmaxf(M, p[i].mx);
        M = warp_max(M);
        double t = 0.0;
        for (int i = lane; i < chunks; i += 32) t += p[i].sum * exp(double(p[i].mx) - double(M));
        t = warp_sum(t);
        if (lane == 0) lse[b] = double(M) + log(t);
        __syncwarp();
        if (chunks <= 64) {
            int h0 = 0, h1 = 0;
            auto head = [&](int i, int h) { return i < chunks && h < k ? c[i * k + h] : 0ull; };
            unsigned long long u0 = head(lane, 0), u1 = head(lane + 32, 0);
            for (int r = 0; r < k; ++r) {
                const unsigned long long best = warp_best(u0 > u1 ? u0 : u1);
                if (lane == 0) best_of[b * k + r] = best;
                if (best && u0 == best) u0 = head(lane, ++h0);
                else if (best && u1 == best) u1 = head(lane + 32, ++h1);
            }
        } else {  // long rows: the next best is the largest below the last
            unsigned long long below = ~0ull;
            for (int r = 0; r < k; ++r) {
                unsigned long long h = 0ull;
                for (int64_t i = lane; i < int64_t(chunks) * k; i += 32) {
                    const unsigned long long u = c[i];
                    if (u < below && u > h) h = u;
                }
                below = warp_best(h);
                if (lane == 0) best_of[b * k + r] = below;
            }
        }
        __syncwarp();
    }
    __syncthreads();
    if (warp) return;
    // over the rows: lane holds rows lane and lane + 32, the score of each one's next candidate as an ordered number (0: none)
    int at[2] = {0, 0};
    unsigned long long next[2];
    auto look = [&](int j) -> unsigned long long {
        const int i = lane + 32 * j;
        const unsigned long long u = i < beams && at[j] < k ? best_of[i * k + at[j]] : 0ull;
        if (!u) return 0ull;
        const double x = scores[int64_t(blockIdx.x) * beams + i] + (double(beam_logit(unsigned(u >> 32))) - lse[i]);
        const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(x));
        return x > -INFINITY && x < INFINITY ? (bits >> 63 ? ~bits : bits | 0x8000000000000000ull) : 0ull;
    };
    next[0] = look(0);
    next[1] = beams > 32 ? look(1) : 0ull;
    for (int r = 0; r < k; ++r) {
        const unsigned long long most = warp_best(next[0] > next[1] ? next[0] : next[1]);
        // equal scores: the lowest row (ballots of rows 0-31, then 32-63; -0 and 0 are equal scores)
        const unsigned a = __ballot_sync(0xffffffffu, most && next[0] == most), b = __ballot_sync(0xffffffffu, most && next[1] == most);
        const int row = a ? __ffs(int(a)) - 1 : b ? 31 + __ffs(int(b)) : -1;
        const int64_t w = int64_t(blockIdx.x) * k + r;
        if (row < 0) {
            if (lane == 0) { score[w] = -INFINITY; parent[w] = -1; token[w] = -1; }
        } else if (lane == (row & 31)) {
            const int j = row >> 5;
            const unsigned long long bits = most >> 63 ? most & 0x7fffffffffffffffull : ~most;
            score[w] = __longlong_as_double(static_cast<long long>(bits));
            parent[w] = int(blockIdx.x) * beams + row;
            token[w] = int(~unsigned(best_of[row * k + at[j]]));
            ++at[j];
            next[j] = look(j);
        }
        __syncwarp();
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
    int groups_log = 3;  // groups of threads: a power of two, k at least, 8 (a warp each) to 64
    while ((1 << groups_log) < k) ++groups_log;
    const bool vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld % 4 == 0;
    const dim3 grid{unsigned(chunks), unsigned(rows)};
    if (vec) k_beam_chunks<true><<<grid, BS_THREADS, 0, s>>>(logits, ld, n_vocab, k, groups_log, allowed, allowed_ld, parts, cand);
    else k_beam_chunks<false><<<grid, BS_THREADS, 0, s>>>(logits, ld, n_vocab, k, groups_log, allowed, allowed_ld, parts, cand);
    ELB_CUDA(cudaGetLastError());
    const size_t smem = (size_t(beams) * k + size_t(BS_WARPS) * BJ_STAGE) * 8;
    ELB_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(k_beam_join), (64 * BS_MAXK + BS_WARPS * BJ_STAGE) * 8));
    ELB_TRY(launch_after(k_beam_join, dim3(unsigned(n_group)), dim3(BS_THREADS), smem, s, true, parts, cand, chunks, beams, k, scores, parent, token, score));
    return ELB_OK;
}

}  // namespace elb
