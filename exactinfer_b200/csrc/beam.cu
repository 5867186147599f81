// Beam search's selection (elb_beam_select_dev): of the candidates (row b, token t) of a group, scored
// d_scores[b] + (x_bt - log sum_u exp x_bu) in double precision, the k best.
//
// Bound by memory: the logits are read once, by k_beam_segments: a warp per segment of 512 logits leaves its maximum, its sum of
// exponentials behind that maximum and the largest logit that may be picked. Everything else works on these: k_beam_pick,
// a block per row, joins the sums, takes a bound that k logits reach from the segments' largest, and reads again only the
// segments that reach it (the order of equal logits needs no care: all at the bound are looked at); the block of a group that comes
// last picks over the rows. (The k best of every 4096 logits, found where they were read, were 2.4 times the instructions.)
// Places are found by counting the larger ones.
//
// Exponentials are the work beside the loads: double precision, e^y = 2^(i/64) 2^n e^r with y = (64 n + i) ln 2 / 64 + r, |r| <= a =
// ln 2 / 128, and the Taylor sum of e^r to the fifth power, whose last term is put into the lower ones by its Chebyshev expansion: r^5 =
// 5/4 a^2 r^3 - 5/16 a^4 r but for a^5 / 16 (e^r is 2.5e-15 off at most; the sum to r^4 / 24 by itself 4e-14), nine double operations a logit. 64 rows of 151936 logits
// in 16 groups under masks: 26.5 us, 17 of them k_beam_segments (65 % of the issue slots, 38 % of the fp64 pipe; bytes alone 6); one group of 4 rows 12 us,
// the length of the two kernels' chains.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "kv.cuh"

namespace elb {

namespace {

constexpr int BS_THREADS = 256, BS_WARPS = 8, BS_PER = 16, BS_SEG = 32 * BS_PER, BS_MAXK = 64;
constexpr int BS_MAXSEG = 2048;  // segments of a row; longer rows have longer ones
constexpr int BP_THREADS = 128, BP_LIST = 1024, BP_SEGS = 8;

struct BeamSeg { double sum; float mx; unsigned top; };  // top: beam_key of the largest logit that may be picked
struct BeamBest { unsigned long long score; int token, pad; };  // score: beam_order

// order of a logit as an unsigned number; 0: not a candidate (-infinity or NaN)
__device__ __forceinline__ unsigned beam_key(float x) {
    const unsigned u = __float_as_uint(x + 0.f);  // (-0 and 0 are equal logits)
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

// 2^(i/64), i << 14 less in the upper word: adding n << 14 to that of entry n & 63 multiplies by the whole powers of two in n / 64
struct BeamTab { unsigned long long e[64]; };
// sum + e^y for -701 <= y <= 0. NaN stays NaN
__device__ __forceinline__ double add_exp(double sum, double y, const double* tab) {
    const double t = fma(y, 92.332482616893656769, 6755399441055744.0);  // 64 / ln 2; 1.5 * 2^52: the low word is the rounded integer
    const double r = fma(t - 6755399441055744.0, -0.010830424696249145, y);  // ln 2 / 64
    const int n = __double2loint(t);
    constexpr double a2 = 0.0054152123481245725 * 0.0054152123481245725;  // (ln 2 / 128)^2
    double p = fma(r, 1.0 / 24.0, 1.0 / 6.0 + a2 / 96.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0 - a2 * a2 / 384.0);
    p = fma(p, r, 1.0);
    const double s = tab[n & 63];
    return fma(__hiloint2double(__double2hiint(s) + n * 16384, __double2loint(s)), p, sum);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// order of a finite score as an unsigned number (0: none)
__device__ __forceinline__ unsigned long long beam_order(double x) {
    const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(x + 0.0));  // (-0 and 0 are equal scores)
    return x > -INFINITY && x < INFINITY ? (bits >> 63 ? ~bits : bits | 0x8000000000000000ull) : 0ull;
}

// grid (segments / 8, rows); VEC: rows start on 16-byte boundaries. `steps` times 512 logits per segment.
template <bool VEC>
__global__ void __launch_bounds__(BS_THREADS, 5) k_beam_segments(const float* __restrict__ logits, int64_t ld, int n, int segs, int steps, int beams,
                                                                 const uint32_t* __restrict__ allowed, int64_t allowed_ld,
                                                                 BeamSeg* __restrict__ parts, unsigned* __restrict__ arrived,
                                                                 const __grid_constant__ BeamTab powers) {
    __shared__ double tab[64];
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, seg = int(blockIdx.x) * BS_WARPS + (tid >> 5);
    const int64_t row = blockIdx.y;
    const float* x = logits + row * ld;
    const uint32_t* mask = allowed ? allowed + row * allowed_ld : nullptr;
    if (blockIdx.x == 0 && tid == 0 && row % beams == 0) arrived[row / beams] = 0;  // for the second launch
    float mx = -INFINITY;
    double sum = 0.0;
    unsigned top = 0;
    for (int st = 0; st < steps; ++st) {
        const int base = (seg * steps + st) * BS_SEG;
        float v[BS_PER];
#pragma unroll
        for (int q = 0; q < BS_PER / 4; ++q) {
            const int i = base + 128 * q + 4 * lane;
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
                const int i = base + 128 * q + 4 * lane;
                off |= (i < n ? ~(mask[i >> 5] >> (i & 31)) & 15u : 15u) << (4 * q);
            }
        }
        if (st == 0) {
            if (tid < 64) tab[tid] = __longlong_as_double(static_cast<long long>(powers.e[tid]));
            __syncthreads();
        }
        float here = -INFINITY;  // (NaN is passed over here and spoils the sum below)
#pragma unroll
        for (int j = 0; j < BS_PER; j += 2) here = max3(here, v[j], v[j + 1]);
        float best = here;
        if (mask) {
            best = -INFINITY;
#pragma unroll
            for (int j = 0; j < BS_PER; j += 2) best = max3(best, (off >> j) & 1u ? -INFINITY : v[j], (off >> j) & 2u ? -INFINITY : v[j + 1]);
        }
        top = max(top, __reduce_max_sync(0xffffffffu, beam_key(best)));
        const unsigned most = __reduce_max_sync(0xffffffffu, beam_key(here));
        here = most ? beam_logit(most) : -INFINITY;
        if (here > mx) {
            sum = mx == -INFINITY ? sum : sum * exp(double(mx) - double(here));
            mx = here;
        }
        // Terms below e^-700 of the largest, and places behind the row's end, count as e^-700: nothing beside the largest's 1
        if (fabsf(mx) >= 16777216.f && mx > -INFINITY) {  // mx - 700 is no fp32 number
            const double from = mx;
#pragma unroll
            for (int j = 0; j < BS_PER; ++j) {
                const double y = double(v[j]) - from;
                sum = add_exp(sum, y < -700.0 ? -700.0 : y, tab);
            }
        } else if (mx > -INFINITY) {
            const float low = mx - 700.f;
            const double from = mx;
#pragma unroll
            for (int j = 0; j < BS_PER; ++j) sum = add_exp(sum, double(max_nan(v[j], low)) - from, tab);
        } else {
#pragma unroll
            for (int j = 0; j < BS_PER; ++j) sum = v[j] != v[j] ? double(NAN) : sum;
        }
    }
    sum = warp_sum(sum);
    if (lane == 0 && seg < segs) parts[row * segs + seg] = BeamSeg{mx < INFINITY ? sum : double(NAN), mx, top};  // (+infinity: no log-sum-exp)
}

// A block per row.
__global__ void __launch_bounds__(BP_THREADS) k_beam_pick(const float* __restrict__ logits, int64_t ld, int n, int segs, int steps, int beams, int k, bool vec,
                                                          const uint32_t* __restrict__ allowed, int64_t allowed_ld,
                                                          const BeamSeg* __restrict__ parts, const double* __restrict__ scores,
                                                          BeamBest* __restrict__ rows_best, unsigned* __restrict__ arrived,
                                                          int* __restrict__ parent, int* __restrict__ token, double* __restrict__ score) {
    constexpr int WARPS = BP_THREADS / 32;
    __shared__ unsigned top[BS_MAXSEG], group_top[32];
    __shared__ unsigned long long list[BP_LIST];
    __shared__ __align__(16) float vals[BP_SEGS * BS_SEG];
    __shared__ int chosen[BS_MAXSEG];
    __shared__ float red_f[WARPS];
    __shared__ double red_d[WARPS];
    __shared__ unsigned long long red_k[WARPS];
    __shared__ int count, some;
    __shared__ bool last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x;
    const float* x = logits + row * ld;
    const uint32_t* mask = allowed ? allowed + row * allowed_ld : nullptr;
    const double own = scores[row];  // (an input of the call: nothing in front of this kernel writes it)
    pdl_wait();
    const BeamSeg* p = parts + row * segs;
    // segments: the row's maximum and sum, and the k with the largest logits, the lower of equal ones first
    const BeamSeg none{0.0, -INFINITY, 0u};
    BeamSeg mine[4];
    float M = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        mine[j] = tid + j * BP_THREADS < segs ? p[tid + j * BP_THREADS] : none;
        if (tid + j * BP_THREADS < segs) top[tid + j * BP_THREADS] = mine[j].top;
        M = fmaxf(M, mine[j].mx);
    }
    for (int i = tid + 4 * BP_THREADS; i < segs; i += BP_THREADS) {
        top[i] = p[i].top;
        M = fmaxf(M, p[i].mx);
    }
    M = warp_max(M);
    if (lane == 0) red_f[warp] = M;
    if (tid == 0) { count = 0; some = 0; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, red_f[w]);
    auto term = [&](const BeamSeg& q) { return q.mx == -INFINITY ? q.sum : q.sum * exp(double(q.mx) - double(M)); };
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += term(mine[j]);
    for (int i = tid + 4 * BP_THREADS; i < segs; i += BP_THREADS) sum += term(p[i]);
    sum = warp_sum(sum);
    if (lane == 0) red_d[warp] = sum;
    // A bound that at least k logits reach: every thread has the largest of its segments; of 32 groups of threads the k-th largest
    // of their maxima (sorted across a warp), for k > 32 the smallest of 64 pairs' maxima.
    unsigned most = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) most = max(most, mine[j].top);
    for (int i = tid + 4 * BP_THREADS; i < segs; i += BP_THREADS) most = max(most, top[i]);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    if (k <= 32) {
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        if ((lane & 3) == 0) group_top[tid / 4] = most;
        __syncthreads();
        unsigned v = group_top[lane];
#pragma unroll 1
        for (int size = 2; size <= 32; size *= 2)
#pragma unroll 1
            for (int d = size / 2; d > 0; d /= 2) {  // descending
                const unsigned o = __shfl_xor_sync(0xffffffffu, v, d);
                v = ((lane & d) == 0) == ((lane & size) == 0) ? max(v, o) : min(v, o);
            }
        most = __shfl_sync(0xffffffffu, v, k - 1);
    } else {
        most = __reduce_min_sync(0xffffffffu, most);
        if (lane == 0) group_top[warp] = most;
        __syncthreads();
        for (int w = 0; w < WARPS; ++w) most = min(most, group_top[w]);
    }
    const unsigned bound = most;
    for (int i = tid; i < segs; i += BP_THREADS) {
        const unsigned u = top[i];
        if (u && u >= bound) chosen[atomicAdd(&some, 1)] = i;
    }
    __syncthreads();
    double lse = 0.0;
    for (int w = 0; w < WARPS; ++w) lse += red_d[w];
    lse = double(M) + log(lse);
    const bool live = lse > -INFINITY && lse < INFINITY && own > -INFINITY && own < INFINITY;
    // their logits once more, eight segments' step at a time
    const int taken = live ? some : 0;
    auto key_at = [&](int c, int st, int e) -> unsigned long long {  // element e of step st of chosen segment c, 0 when it is no candidate
        const int i = (chosen[c] * steps + st) * BS_SEG + e;
        const unsigned key = i < n && (!mask || ((mask[i >> 5] >> (i & 31)) & 1u)) ? beam_key(__ldcg(x + i)) : 0u;
        return key >= bound ? beam_pack(key, i) : 0ull;
    };
    for (int st = 0; st < steps; ++st)
        for (int c0 = 0; c0 < taken; c0 += BP_SEGS) {
            const int here = min(BP_SEGS, taken - c0);
            for (int e = 4 * tid; e < here * BS_SEG; e += 4 * BP_THREADS) {
                const int i = (chosen[c0 + e / BS_SEG] * steps + st) * BS_SEG + e % BS_SEG;
                if (vec && i + 3 < n) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(vals + e))), "l"(x + i) : "memory");
                } else {
                    for (int q = 0; q < 4; ++q) vals[e + q] = i + q < n ? __ldcg(x + i + q) : -INFINITY;
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            const float low = bound ? beam_logit(bound) : -INFINITY;
            for (int e = 4 * tid; e < here * BS_SEG; e += 4 * BP_THREADS) {  // (a thread's own)
                const float4 v = *reinterpret_cast<const float4*>(vals + e);
                const float most = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
                if (!(most >= low) || most == -INFINITY) continue;
                for (int q = 0; q < 4; ++q) {
                    const float w = vals[e + q];
                    const int i = (chosen[c0 + e / BS_SEG] * steps + st) * BS_SEG + e % BS_SEG + q;
                    if (!(w >= low) || w == -INFINITY || (mask && !((mask[i >> 5] >> (i & 31)) & 1u))) continue;
                    const int at = atomicAdd(&count, 1);  // (the order does not matter: places are counted)
                    if (at < BP_LIST) list[at] = beam_pack(beam_key(w), i);
                }
            }
        }
    __syncthreads();
    BeamBest* mine_best = rows_best + row * k;
    const int have = count;
    auto put = [&](int place, unsigned long long u) {
        mine_best[place] = BeamBest{u ? beam_order(own + (double(beam_logit(unsigned(u >> 32))) - lse)) : 0ull, int(~unsigned(u)), 0};
    };
    if (have <= BP_LIST) {
        for (int c = tid; c < have; c += BP_THREADS) {
            const unsigned long long me = list[c];
            int place = 0;
#pragma unroll 8
            for (int o = 0; o < have; ++o) place += list[o] > me;
            if (place < k) put(place, me);
        }
        for (int r = have + tid; r < k; r += BP_THREADS) put(r, 0ull);
    } else {  // many logits at the bound (equal ones): one after the other
        unsigned long long below = ~0ull;
        for (int r = 0; r < k; ++r) {
            unsigned long long h = 0ull;
            for (int st = 0; st < steps; ++st)
                for (int e = tid; e < taken * BS_SEG; e += BP_THREADS) {
                    const unsigned long long u = key_at(e / BS_SEG, st, e % BS_SEG);
                    if (u < below && u > h) h = u;
                }
            h = warp_best(h);
            if (lane == 0) red_k[warp] = h;
            __syncthreads();
            below = 0ull;
            for (int w = 0; w < WARPS; ++w) below = red_k[w] > below ? red_k[w] : below;
            if (tid == 0) put(r, below);
            __syncthreads();
        }
    }
    // the group's last block picks over its rows
    __threadfence();
    __syncthreads();
    const int64_t group = row / beams;
    if (tid == 0) last = atomicAdd(arrived + group, 1u) == unsigned(beams - 1);
    __syncthreads();
    if (!last) return;
    __threadfence();
    const BeamBest* best = rows_best + group * beams * k;
    const int all = beams * k;
    for (int i = tid; i < min(all, BP_LIST); i += BP_THREADS) list[i] = __ldcg(&best[i].score);
    for (int r = tid; r < k; r += BP_THREADS) { score[group * k + r] = -INFINITY; parent[group * k + r] = -1; token[group * k + r] = -1; }
    __syncthreads();
    // (score, then row, then rank within the row: i = row * k + rank)
    for (int i = tid; i < all; i += BP_THREADS) {
        const unsigned long long me = i < BP_LIST ? list[i] : __ldcg(&best[i].score);
        if (!me) continue;
        int place = 0;
#pragma unroll 4
        for (int o = 0; o < min(all, BP_LIST); ++o) place += int(list[o] > me) + (int(list[o] == me) & int(o < i));
        for (int o = BP_LIST; o < all && place < k; ++o) {
            const unsigned long long u = __ldcg(&best[o].score);
            place += int(u > me) + (int(u == me) & int(o < i));
        }
        if (place >= k) continue;
        const unsigned long long bits = me >> 63 ? me & 0x7fffffffffffffffull : ~me;
        score[group * k + place] = __longlong_as_double(static_cast<long long>(bits));
        parent[group * k + place] = int(group) * beams + i / k;
        token[group * k + place] = __ldcg(&best[i].token);
    }
}

// segments of a row and their length in steps of 512 logits
struct BeamCut { int segs, steps; };
BeamCut beam_cut(int n) {
    const int64_t all = (int64_t(n) + BS_SEG - 1) / BS_SEG;
    const int steps = int((all + BS_MAXSEG - 1) / BS_MAXSEG);
    return BeamCut{int((all + steps - 1) / steps), steps};
}
size_t up256(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace

size_t beam_select_work(int n_vocab, int n_group, int beams, int k) {
    if (n_vocab <= 0 || n_vocab > (1 << 30) || n_group < 0 || beams <= 0 || beams > 64 || k <= 0 || k > BS_MAXK || int64_t(n_group) * beams > 65535) return 0;
    const size_t rows = size_t(n_group) * beams;
    return std::max<size_t>(256, up256(rows * size_t(beam_cut(n_vocab).segs) * sizeof(BeamSeg)) + up256(rows * k * sizeof(BeamBest)) + up256(size_t(n_group) * 4));
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
    // A row's block reads its score at its start, and a group's results come behind all of its rows: in place they may only stand
    // where the group's own scores do.
    const uintptr_t s0 = reinterpret_cast<uintptr_t>(scores), r0 = reinterpret_cast<uintptr_t>(score);
    const size_t rows_bytes = size_t(n_group) * beams * sizeof(double), picks = size_t(n_group) * k;
    auto touches = [&](const void* p, size_t n) { const uintptr_t x = reinterpret_cast<uintptr_t>(p); return x < s0 + rows_bytes && s0 < x + n; };
    if (touches(parent, picks * 4) || touches(token, picks * 4) || (touches(score, picks * 8) && !(s0 == r0 && k == beams)))
        return fail(ELB_ERR_INVALID, "beam_select: outputs must not overlap the scores (d_score may be d_scores when k = beams)");
    const int rows = n_group * beams;
    const BeamCut cut = beam_cut(n_vocab);
    uint8_t* at = static_cast<uint8_t*>(work);
    auto* parts = reinterpret_cast<BeamSeg*>(at);
    at += up256(size_t(rows) * cut.segs * sizeof(BeamSeg));
    auto* best = reinterpret_cast<BeamBest*>(at);
    at += up256(size_t(rows) * k * sizeof(BeamBest));
    auto* arrived = reinterpret_cast<unsigned*>(at);
    const bool vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld % 4 == 0;
    const dim3 grid{unsigned((cut.segs + BS_WARPS - 1) / BS_WARPS), unsigned(rows)};
    static const BeamTab powers = [] {
        BeamTab t;
        for (int i = 0; i < 64; ++i) {
            const double e = std::exp2(i / 64.0);
            std::memcpy(t.e + i, &e, sizeof e);
            t.e[i] -= static_cast<unsigned long long>(i << 14) << 32;
        }
        return t;
    }();
    if (vec) k_beam_segments<true><<<grid, BS_THREADS, 0, s>>>(logits, ld, n_vocab, cut.segs, cut.steps, beams, allowed, allowed_ld, parts, arrived, powers);
    else k_beam_segments<false><<<grid, BS_THREADS, 0, s>>>(logits, ld, n_vocab, cut.segs, cut.steps, beams, allowed, allowed_ld, parts, arrived, powers);
    ELB_CUDA(cudaGetLastError());
    ELB_TRY(launch_after(k_beam_pick, dim3(unsigned(rows)), dim3(BP_THREADS), 0, s, true, logits, ld, n_vocab, cut.segs, cut.steps, beams, k, vec, allowed,
                         allowed_ld, parts, scores, best, arrived, parent, token, score));
    return ELB_OK;
}

}  // namespace elb
