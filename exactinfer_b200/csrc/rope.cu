// Rotary positions, alone (elb_rope_dev) and on the way into the pages of a cache (elb_kv_append_dev): per head an optional
// RMSNorm x * (1 / sqrt(mean x^2 + eps)) * w (src/ops.cpp:155-160 of the reference, sum of squares in double), then pair i
// of the first `dim` values turned by pos * f_i and multiplied by m (src/model.cpp:23-32 with its scaled forms).
//
// Bound by memory: every value is read and written once. A block takes a few tokens, computes the cosines and sines that
// all their heads share once, in double, into shared memory, and streams the heads through registers: a thread takes 8
// values (a "unit": 4 pairs, or 8 values that are kept) as two 16-byte quads. Angles are formed in turns, t = pos * (f / 2 pi) and
// the fraction of t, so that no position needs more than one double-precision product and a sine of at most one turn.
// 4096 rows of 32 heads of 128, interleaved: 23.5 us, 5.7 TB/s (26.7 with a thread's eight values side by side: every load and
// store touched half of its sectors). Append of 2048 tokens, 64 + 8 + 8 heads, F16: 37.2 us, 4.3 TB/s: one wave of blocks, whose first
// loads wait beside the search for their tokens and the angles.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "kv.cuh"

namespace elb {

namespace {

constexpr int RP_THREADS = 256, RP_TOKENS = 4, RP_MAXHALF = 128, RP_BATCH = 4, RP_PAIRS = 256;

struct RopeArgs {
    const double* turns;  // [half] or null: no rotation
    int dim, layout, head_dim;
    float mscale, eps;
    // queries: n_head heads of row t at q + t * ldq -> q_out + t * ldqo
    const float* q;
    float* q_out;
    const float* q_norm;
    int64_t ldq, ldqo;
    int n_head;
    // keys and values into pages (HKV = 0: none)
    const float *k, *v, *k_norm;
    int64_t ldk, ldv;
    int HKV, planes;
    __half* pool;  // this layer
    int64_t n;
    const int* pos;  // positions of the rows, or null: from the batch
    KvRows rows;
};

// 1 / sqrt(ms) for a mean square in double: an fp32 estimate and one Newton step (2^-44), double division outside fp32's range
__device__ __forceinline__ float inv_rms(double ms) {
    if (!(ms > 1e-30 && ms < 1e30)) return float(1.0 / sqrt(ms));
    const double y = rsqrtf(float(ms));
    return float(y * (1.5 - 0.5 * ms * y * y));
}

// four values -> the fp16 planes of a pool row (lo plane: `plane` halves behind); the remainder of an infinity is 0
__device__ __forceinline__ void store4(__half* dst, int planes, int64_t plane, const float* v) {
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        hi[i] = *reinterpret_cast<const uint32_t*>(&h);
        if (planes == 2) {
            const float2 f = __half22float2(h);
            const __half2 l = __floats2half2_rn(isinf(f.x) ? 0.f : v[2 * i] - f.x, isinf(f.y) ? 0.f : v[2 * i + 1] - f.y);
            lo[i] = *reinterpret_cast<const uint32_t*>(&l);
        }
    }
    *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
    if (planes == 2) *reinterpret_cast<uint2*>(dst + plane) = make_uint2(lo[0], lo[1]);
}

// What a block knows of one of its tokens
struct Tok {
    int pos;      // position
    int on;       // there is such a row and it belongs to a sequence
    int64_t row;  // halves from the layer's first to the token's first in its page (kv 0, head 0), or -1: not stored
};

// Positions and page rows of the block's tokens. Batch: sequence s holds row t when q_start[s] <= t < q_start[s + 1]; all threads
// look, one finds it (of overlapping ranges the last counts).
__device__ __forceinline__ void find_tokens(const RopeArgs& a, int64_t t0, int tokens, Tok* tok, int* seq) {
    const int tid = threadIdx.x;
    if (a.pos) {
        if (tid < tokens) tok[tid] = Tok{t0 + tid < a.n ? a.pos[t0 + tid] : 0, t0 + tid < a.n, -1};
        __syncthreads();
        return;
    }
    if (tid < tokens) seq[tid] = -1;
    __syncthreads();
    for (int s = tid; s < a.rows.n_seq; s += RP_THREADS) {
        const int lo = a.rows.q_start[s], hi = a.rows.q_start[s + 1];
        for (int i = 0; i < tokens; ++i)
            if (lo <= t0 + i && t0 + i < hi && t0 + i < a.n) atomicMax(seq + i, s);
    }
    __syncthreads();
    if (tid < tokens) {
        Tok t{0, 0, -1};
        if (seq[tid] >= 0) {
            const KvSeq q = kv_seq(a.rows, seq[tid]);
            t.pos = q.len - q.nq + int(t0 + tid - q.row0);
            t.on = t.pos >= 0;
            const int pg = kv_page(a.rows, seq[tid], t.pos);
            if (t.on && pg >= 0) t.row = (int64_t(pg) * 2 * a.HKV * a.planes * a.rows.page + (t.pos & (a.rows.page - 1))) * KV_D;
        }
        tok[tid] = t;
    }
    __syncthreads();
}

// PERM: pairs 4 u, 4 u + 1 of all u first, then 4 u + 2, 4 u + 3: lanes that each read four pairs in two 16-byte loads meet no conflicts
template <bool PERM> __device__ __forceinline__ void fill_angles(const RopeArgs& a, int tokens, const Tok* tok, float2 (*cs)[RP_MAXHALF]) {
    const int half = a.dim / 2;
    for (int i = threadIdx.x; i < tokens * half; i += RP_THREADS) {
        const int t = i / half, f = i - t * half;
        const double turn = double(tok[t].pos) * a.turns[f];
        double sn, c;
        sincospi(2.0 * (turn - rint(turn)), &sn, &c);
        cs[t][PERM ? (f >> 2) * 2 + (f & 2) * (RP_MAXHALF / 4) + (f & 1) : f] = make_float2(float(c * a.mscale), float(sn * a.mscale));
    }
}

// A (token, head) pair of a block: where it comes from (null: nowhere) and goes to (0: nowhere), its kind (0: queries, 1: keys, 2:
// values) in the address's lowest two bits and the token's number in the next two (rows start on 16-byte boundaries)
struct Pair { const float* src; unsigned long long dst; };

__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
    const float x0 = x, y0 = y;
    x = x0 * c - y0 * s;
    y = x0 * s + y0 * c;
}

// head_dim 32, 64, 128 or 256 (2^upt_log units), dim a multiple of 8, rows on 16-byte boundaries; grid (token groups, head groups).
// Thread: unit u of every slots-th pair of the block, RP_BATCH pairs at a time, whose loads go out together - the first ones before
// the block knows its tokens. Addresses are worked out once per pair, into shared memory (by every thread for itself they were 40
// % of the instructions), and a thread's place in a head is the same for all pairs: values, which are not turned, are read and
// written in the pairs' order too.
template <bool NORM, bool HALF>
__global__ void __launch_bounds__(RP_THREADS, 4) k_rope(const RopeArgs a, int tokens, int heads_per_block, int upt_log) {
    __shared__ __align__(16) float2 cs[RP_TOKENS][RP_MAXHALF];
    __shared__ __align__(16) float weights[NORM ? 2 : 1][NORM ? 2 * RP_MAXHALF : 4];  // of queries, keys
    __shared__ __align__(16) Pair pair[RP_PAIRS];
    __shared__ Tok tok[RP_TOKENS];
    __shared__ int seq[RP_TOKENS];
    const int64_t t0 = int64_t(blockIdx.x) * tokens;
    const int heads = a.n_head + 2 * a.HKV, h0 = blockIdx.y * heads_per_block, nh = min(heads_per_block, heads - h0);
    const int upt = 1 << upt_log, u = threadIdx.x & (upt - 1), slot = threadIdx.x >> upt_log, slots = RP_THREADS >> upt_log;
    const int pairs = tokens * nh;
    const double part = 1.0 / double(1 << (upt_log + 3));  // 1 / head_dim, exact
    // a thread's two quads of a head: pairs' halves, or two pairs each
    const bool both = a.turns && 8 * u < a.dim;
    const int e0 = HALF ? (both ? 4 * u : 8 * u) : 4 * u, e1 = HALF ? (both ? a.dim / 2 + 4 * u : 8 * u + 4) : 4 * u + a.head_dim / 2;
    const bool turn0 = HALF ? both : a.turns && e0 < a.dim, turn1 = HALF ? both : a.turns && e1 < a.dim;
    for (int p = threadIdx.x; p < pairs; p += RP_THREADS) {
        const int tt = p / nh, h = h0 + p - tt * nh, hk = h - a.n_head, hv = hk - a.HKV;
        const int64_t t = t0 + tt;
        pair[p].src = t >= a.n ? nullptr : hv >= 0 ? a.v + t * a.ldv + hv * KV_D : hk >= 0 ? a.k + t * a.ldk + hk * KV_D
                                                                                           : a.q + t * a.ldq + int64_t(h) * a.head_dim;
    }
    if (NORM)
        for (int i = threadIdx.x; i < a.head_dim; i += RP_THREADS) {
            if (a.q_norm) weights[0][i] = a.q_norm[i];
            if (a.k_norm) weights[NORM][i] = a.k_norm[i];
        }
    __syncthreads();
    for (int p0 = slot; p0 - slot < pairs; p0 += RP_BATCH * slots) {  // (whole warps stay together for the reductions)
        float v[RP_BATCH][8];
#pragma unroll
        for (int b = 0; b < RP_BATCH; ++b) {
            const int p = p0 + b * slots;
            const float* src = p < pairs ? pair[p].src : nullptr;
            if (src) {
                *reinterpret_cast<float4*>(v[b]) = __ldcg(reinterpret_cast<const float4*>(src + e0));
                *reinterpret_cast<float4*>(v[b] + 4) = __ldcg(reinterpret_cast<const float4*>(src + e1));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[b][i] = 0.f;
            }
        }
        if (p0 == slot) {
            find_tokens(a, t0, tokens, tok, seq);
            if (a.turns) fill_angles<HALF>(a, tokens, tok, cs);
            for (int p = threadIdx.x; p < pairs; p += RP_THREADS) {
                const int tt = p / nh, h = h0 + p - tt * nh, hk = h - a.n_head, is_v = hk >= a.HKV;
                unsigned long long to = 0;
                if (hk < 0) {
                    if (tok[tt].on) to = reinterpret_cast<unsigned long long>(a.q_out + (t0 + tt) * a.ldqo + int64_t(h) * a.head_dim);
                } else if (tok[tt].on && tok[tt].row >= 0) {
                    to = reinterpret_cast<unsigned long long>(a.pool + tok[tt].row + int64_t(hk) * a.planes * a.rows.page * KV_D) | (1 + is_v);
                }
                pair[p].dst = to ? to | unsigned(tt << 2) : 0ull;
            }
            __syncthreads();
        }
        // Mean squares of the batch's four heads at once: the first two steps of the reduction across a head's lanes halve what a
        // lane holds, so that it ends with one head's sum, and every lane forms one factor
        float inv = 1.f;
        if (NORM) {
            static_assert(RP_BATCH == 4, "two halving steps");
            double ss[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                ss[b] = 0.0;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss[b] = fma(double(v[b][i]), double(v[b][i]), ss[b]);
            }
            const bool odd = u & 1, third = u & 2;
            const double k0 = odd ? ss[2] : ss[0], k1 = odd ? ss[3] : ss[1], g0 = odd ? ss[0] : ss[2], g1 = odd ? ss[1] : ss[3];
            const double a0 = k0 + __shfl_xor_sync(0xffffffffu, g0, 1), a1 = k1 + __shfl_xor_sync(0xffffffffu, g1, 1);
            double sum = (third ? a1 : a0) + __shfl_xor_sync(0xffffffffu, third ? a0 : a1, 2);
            for (int o = 4; o < upt; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            inv = inv_rms(sum * part + double(a.eps));  // of head 2 (u & 1) + (u / 2 & 1)
        }
#pragma unroll
        for (int b = 0; b < RP_BATCH; ++b) {
            const int p = p0 + b * slots;
            const float mine = NORM ? __shfl_sync(0xffffffffu, inv, (int(threadIdx.x) & 31 & ~3) | (b >> 1) | (b & 1) << 1) : 1.f;
            const unsigned long long to = p < pairs ? pair[p].dst : 0ull;
            if (!to) continue;
            const unsigned kind = unsigned(to) & 3u, t = unsigned(to) >> 2 & 3u;
            if (NORM && kind < 2 && (kind ? a.k_norm : a.q_norm)) {
                const float4 w0 = *reinterpret_cast<const float4*>(weights[kind] + e0), w1 = *reinterpret_cast<const float4*>(weights[kind] + e1);
                const float ww[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) v[b][i] = __fmul_rn(__fmul_rn(v[b][i], mine), ww[i]);
            }
            if (turn0 && kind < 2) {
                const float4* c = reinterpret_cast<const float4*>(cs[t]) + u;
                if (HALF) {
                    const float4 c0 = c[0], c1 = c[RP_MAXHALF / 4];
                    turn(v[b][0], v[b][4], c0.x, c0.y);
                    turn(v[b][1], v[b][5], c0.z, c0.w);
                    turn(v[b][2], v[b][6], c1.x, c1.y);
                    turn(v[b][3], v[b][7], c1.z, c1.w);
                } else {
                    const float4 c0 = c[0];
                    turn(v[b][0], v[b][1], c0.x, c0.y);
                    turn(v[b][2], v[b][3], c0.z, c0.w);
                    if (turn1) {
                        const float4 c1 = c[upt];
                        turn(v[b][4], v[b][5], c1.x, c1.y);
                        turn(v[b][6], v[b][7], c1.z, c1.w);
                    }
                }
            }
            const unsigned long long at = to & ~15ull;
            if (kind == 0) {
                float* dst = reinterpret_cast<float*>(at);
                *reinterpret_cast<float4*>(dst + e0) = *reinterpret_cast<const float4*>(v[b]);
                *reinterpret_cast<float4*>(dst + e1) = *reinterpret_cast<const float4*>(v[b] + 4);
            } else {
                __half* dst = reinterpret_cast<__half*>(at);
                store4(dst + e0, a.planes, int64_t(a.rows.page) * KV_D, v[b]);
                store4(dst + e1, a.planes, int64_t(a.rows.page) * KV_D, v[b] + 4);
            }
        }
    }
}

// any even head_dim and dim, any alignment: a warp per (row, head), pair by pair
__global__ void __launch_bounds__(RP_THREADS) k_rope_any(const RopeArgs a) {
    __shared__ float2 cs[RP_TOKENS][RP_MAXHALF];
    __shared__ Tok tok[RP_TOKENS];
    __shared__ int seq[RP_TOKENS];
    const int64_t t0 = blockIdx.x;
    find_tokens(a, t0, 1, tok, seq);
    fill_angles<false>(a, 1, tok, cs);
    __syncthreads();
    const int lane = threadIdx.x & 31, half = a.dim / 2;
    for (int h = int(threadIdx.x) / 32 + 8 * int(blockIdx.y); h < a.n_head; h += 8 * int(gridDim.y)) {
        const float* x = a.q + t0 * a.ldq + int64_t(h) * a.head_dim;
        float* y = a.q_out + t0 * a.ldqo + int64_t(h) * a.head_dim;
        float inv = 1.f;
        if (a.q_norm) {
            double ss = 0.0;
            for (int i = lane; i < a.head_dim; i += 32) ss += double(x[i]) * double(x[i]);
            inv = inv_rms(warp_sum(ss) / a.head_dim + double(a.eps));
        }
        auto get = [&](int i) { return a.q_norm ? __fmul_rn(__fmul_rn(x[i], inv), a.q_norm[i]) : x[i]; };
        for (int i = lane; i < half; i += 32) {
            const int i0 = a.layout == ELB_ROPE_HALF ? i : 2 * i, i1 = a.layout == ELB_ROPE_HALF ? i + half : 2 * i + 1;
            const float2 c = cs[0][i];
            const float u = get(i0), v = get(i1);
            y[i0] = u * c.x - v * c.y;
            y[i1] = u * c.y + v * c.x;
        }
        for (int i = a.dim + lane; i < a.head_dim; i += 32) y[i] = get(i);
    }
}

bool aligned16(const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 4 == 0; }

int rope_run(RopeArgs& a, cudaStream_t s) {
    // tokens of a block share its start-up (angles in double): four when there are enough tokens to fill the GPU all the same.
    // Heads are cut over blocks while the grid is small
    const int heads = a.n_head + 2 * a.HKV, tokens = a.n >= 1024 ? 4 : a.n >= 512 ? 2 : 1;
    const int64_t groups = (a.n + tokens - 1) / tokens;
    int cuts = (heads * tokens + RP_PAIRS - 1) / RP_PAIRS, per = (heads + cuts - 1) / cuts;
    while (per > 16 && groups * ((heads + per - 1) / per) < 296) per = (per + 1) / 2;
    int upt_log = 2;
    while ((8 << upt_log) < a.head_dim) ++upt_log;
    const dim3 grid{unsigned(groups), unsigned((heads + per - 1) / per)};
    const bool norm = a.q_norm || a.k_norm, half = a.layout == ELB_ROPE_HALF;
    const auto kernel = norm ? (half ? k_rope<true, true> : k_rope<true, false>) : (half ? k_rope<false, true> : k_rope<false, false>);
    kernel<<<grid, RP_THREADS, 0, s>>>(a, tokens, per, upt_log);
    ELB_CUDA(cudaGetLastError());
    return ELB_OK;
}

}  // namespace

int rope_frequencies(const elb_rope_config* c, std::vector<double>* freq, double* m) {
    if (!c) return fail(ELB_ERR_INVALID, "rope: null configuration");
    if (c->head_dim < 2 || c->head_dim > 256 || c->head_dim % 2 || c->dim < 2 || c->dim > c->head_dim || c->dim % 2)
        return fail(ELB_ERR_INVALID, "rope: head_dim must be even and at most 256, dim even and at most head_dim");
    if (c->layout != ELB_ROPE_HALF && c->layout != ELB_ROPE_INTERLEAVED) return fail(ELB_ERR_INVALID, "rope: unknown layout");
    if (c->scaling < ELB_ROPE_PLAIN || c->scaling > ELB_ROPE_BANDS) return fail(ELB_ERR_INVALID, "rope: unknown scaling");
    if (!(c->base > 1.0) || !std::isfinite(c->base)) return fail(ELB_ERR_INVALID, "rope: base must be finite and above 1");
    if (c->scaling != ELB_ROPE_PLAIN && (!(c->factor >= 1.0) || !std::isfinite(c->factor))) return fail(ELB_ERR_INVALID, "rope: factor must be finite and at least 1");
    const bool yarn = c->scaling == ELB_ROPE_YARN, bands = c->scaling == ELB_ROPE_BANDS;
    if ((yarn || bands) && (!(c->orig_ctx > 0.0) || !std::isfinite(c->orig_ctx))) return fail(ELB_ERR_INVALID, "rope: orig_ctx must be positive");
    if (yarn && (!(c->beta_slow > 0.0) || !(c->beta_fast >= c->beta_slow) || !std::isfinite(c->beta_fast) || !(c->attn_factor >= 0.0) || !std::isfinite(c->attn_factor)))
        return fail(ELB_ERR_INVALID, "rope: beta_fast >= beta_slow > 0 and attn_factor >= 0 are needed");
    if (bands && (!(c->low_freq > 0.0) || !(c->high_freq > c->low_freq) || !std::isfinite(c->high_freq)))
        return fail(ELB_ERR_INVALID, "rope: high_freq > low_freq > 0 is needed");
    const double pi = 3.14159265358979323846, dim = c->dim;
    double lo = 0.0, hi = 0.0;
    *m = 1.0;
    if (yarn) {
        auto at = [&](double turns) { return dim * std::log(c->orig_ctx / (2.0 * pi * turns)) / (2.0 * std::log(c->base)); };
        lo = std::max(std::floor(at(c->beta_fast)), 0.0);
        hi = std::min(std::ceil(at(c->beta_slow)), dim - 1.0);
        if (lo == hi) hi += 0.001;
        *m = c->attn_factor > 0.0 ? c->attn_factor : 0.1 * std::log(c->factor) + 1.0;
    }
    freq->resize(size_t(c->dim / 2));
    for (int i = 0; i < c->dim / 2; ++i) {
        double f = std::pow(c->base, -2.0 * i / dim);
        if (c->scaling == ELB_ROPE_LINEAR) {
            f /= c->factor;
        } else if (yarn) {
            const double r = std::min(std::max((i - lo) / (hi - lo), 0.0), 1.0);
            f = f / c->factor * r + f * (1.0 - r);
        } else if (bands) {
            const double turns = c->orig_ctx * f / (2.0 * pi);
            if (turns < c->low_freq) {
                f /= c->factor;
            } else if (turns <= c->high_freq) {
                const double t = (turns - c->low_freq) / (c->high_freq - c->low_freq);
                f = (1.0 - t) * f / c->factor + t * f;
            }
        }
        (*freq)[size_t(i)] = f;
    }
    return ELB_OK;
}

int rope_create(int device, const elb_rope_config* c, Rope** out) {
    std::vector<double> freq;
    double m = 1.0;
    if (!out) return fail(ELB_ERR_INVALID, "rope_create: null argument");
    ELB_TRY(rope_frequencies(c, &freq, &m));
    DeviceScope on(device);
    if (on.rc != ELB_OK) return on.rc;
    for (double& f : freq) f /= 2.0 * 3.14159265358979323846;
    auto* r = new (std::nothrow) Rope;
    if (!r) return fail(ELB_ERR_MEMORY, "rope_create: out of memory");
    r->device = device; r->head_dim = c->head_dim; r->dim = c->dim; r->layout = c->layout; r->mscale = float(m);
    if (device_malloc(&r->d_turns, freq.size() * sizeof(double)) != cudaSuccess) {
        delete r;
        return fail(ELB_ERR_MEMORY, "rope_create: out of device memory");
    }
    cudaError_t e = cudaMemcpy(r->d_turns, freq.data(), freq.size() * sizeof(double), cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);  // (pageable memory: the copy returns once it is staged)
    if (e != cudaSuccess) {
        rope_destroy(r);
        return fail(ELB_ERR_CUDA, std::string("rope_create: ") + cudaGetErrorString(e));
    }
    *out = r;
    return ELB_OK;
}

void rope_destroy(Rope* r) {
    if (!r) return;
    DeviceScope on(r->device);
    cudaFree(r->d_turns);
    delete r;
}

int rope_launch(const Rope* r, const float* x, int64_t ldx, float* y, int64_t ldy, int64_t n, int heads, const int* pos, const float* norm,
                float eps, cudaStream_t s) {
    if (!r) return fail(ELB_ERR_INVALID, "rope: null handle");
    if (n < 0 || heads <= 0 || heads > 65536) return fail(ELB_ERR_INVALID, "rope: bad row or head count");
    if (n == 0) return ELB_OK;
    if (!x || !y || !pos) return fail(ELB_ERR_INVALID, "rope: null argument");
    const int64_t width = int64_t(heads) * r->head_dim;
    if (ldx < width || ldy < width) return fail(ELB_ERR_INVALID, "rope: a row stride is shorter than the row");
    if (x == y && ldx != ldy) return fail(ELB_ERR_INVALID, "rope: in place needs equal strides");
    if (x != y && rows_meet(x, ldx, width, y, ldy, width, n)) return fail(ELB_ERR_INVALID, "rope: the result must not overlap the input, or must be in its place");
    if (n > 0x7fffffff) return fail(ELB_ERR_UNSUPPORTED, "rope: too many rows");
    if (norm && !(eps >= 0.f)) return fail(ELB_ERR_INVALID, "rope: eps must not be negative");
    DeviceScope on(r->device);
    if (on.rc != ELB_OK) return on.rc;
    RopeArgs a{};
    a.turns = r->d_turns; a.dim = r->dim; a.layout = r->layout; a.head_dim = r->head_dim; a.mscale = r->mscale; a.eps = eps;
    a.q = x; a.q_out = y; a.q_norm = norm; a.ldq = ldx; a.ldqo = ldy; a.n_head = heads; a.n = n; a.pos = pos;
    const int d = r->head_dim;
    if ((d == 32 || d == 64 || d == 128 || d == 256) && r->dim % 8 == 0 && aligned16(x, ldx) && aligned16(y, ldy) && aligned16(norm, 0)) return rope_run(a, s);
    k_rope_any<<<dim3(unsigned(n), unsigned(std::min((heads + 7) / 8, n < 512 ? 8 : 1))), RP_THREADS, 0, s>>>(a);
    ELB_CUDA(cudaGetLastError());
    return ELB_OK;
}

int kv_append_launch(Kv* kv, int layer, const elb_kv_batch* b, const Rope* rope, const float* k, int64_t ldk, const float* v, int64_t ldv,
                     const float* k_norm, float eps, const float* q, int64_t ldq, int n_head, const float* q_norm, float* q_out, int64_t ldqo,
                     cudaStream_t s) {
    ELB_TRY(kv_check_batch(kv, layer, b, "kv_append"));
    if (!k || !v) return fail(ELB_ERR_INVALID, "kv_append: null argument");
    const int64_t kd = int64_t(kv->HKV) * KV_D;
    if (ldk < kd || ldv < kd) return fail(ELB_ERR_INVALID, "kv_append: a row stride is shorter than the row");
    if (!aligned16(k, ldk) || !aligned16(v, ldv)) return fail(ELB_ERR_UNSUPPORTED, "kv_append: rows must start on 16-byte boundaries");
    if (q) {
        if (n_head <= 0 || n_head > 65536 || !q_out) return fail(ELB_ERR_INVALID, "kv_append: queries need their head count and an output");
        if (ldq < int64_t(n_head) * KV_D || ldqo < int64_t(n_head) * KV_D) return fail(ELB_ERR_INVALID, "kv_append: a row stride is shorter than the row");
        if (q == q_out && ldq != ldqo) return fail(ELB_ERR_INVALID, "kv_append: in place needs equal strides");
        if (!aligned16(q, ldq) || !aligned16(q_out, ldqo)) return fail(ELB_ERR_UNSUPPORTED, "kv_append: rows must start on 16-byte boundaries");
    }
    if ((k_norm || (q && q_norm)) && !(eps >= 0.f)) return fail(ELB_ERR_INVALID, "kv_append: eps must not be negative");
    if (!aligned16(k_norm, 0) || (q && !aligned16(q_norm, 0))) return fail(ELB_ERR_UNSUPPORTED, "kv_append: norm weights must start on a 16-byte boundary");
    if (rope && (rope->head_dim != KV_D || rope->device != kv->device)) return fail(ELB_ERR_INVALID, "kv_append: the positions are for another head_dim or device");
    if (rope && rope->dim % 8) return fail(ELB_ERR_UNSUPPORTED, "kv_append: the rotated part of a head must be a multiple of 8");
    if (b->n_tok == 0 || b->n_seq == 0) return ELB_OK;
    const int64_t qd = int64_t(n_head) * KV_D;
    if (q && ((q != q_out && rows_meet(q, ldq, qd, q_out, ldqo, qd, b->n_tok)) || rows_meet(k, ldk, kd, q_out, ldqo, qd, b->n_tok) ||
              rows_meet(v, ldv, kd, q_out, ldqo, qd, b->n_tok)))
        return fail(ELB_ERR_INVALID, "kv_append: the rotated queries must not overlap the inputs, or must be in the queries' place");
    DeviceScope on(kv->device);
    if (on.rc != ELB_OK) return on.rc;
    RopeArgs a{};
    if (rope) { a.turns = rope->d_turns; a.dim = rope->dim; a.layout = rope->layout; a.mscale = rope->mscale; }
    a.head_dim = KV_D; a.eps = eps;
    a.n_head = q ? n_head : 0; a.q = q; a.q_out = q_out; a.q_norm = q ? q_norm : nullptr; a.ldq = ldq; a.ldqo = ldqo;
    a.k = k; a.v = v; a.k_norm = k_norm; a.ldk = ldk; a.ldv = ldv; a.HKV = kv->HKV; a.planes = kv->planes;
    a.pool = kv->mem + int64_t(layer) * kv->layer_halves();
    a.n = b->n_tok; a.rows = kv_rows(kv, b);
    return rope_run(a, s);
}

}  // namespace elb
