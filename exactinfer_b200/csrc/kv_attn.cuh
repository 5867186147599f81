// Attention over a paged cache: what its two kernels and the joining of their partial results share.
#pragma once

#include <algorithm>

#include "kv.cuh"

namespace elb {

struct KvAttnArgs {
    KvRows rows;
    const __half* pool;  // this layer
    const float* q;
    float* out;
    int64_t ldq, ldo;
    int H, HKV, group, planes;
    float scale2;        // scale * log2(e): weights are powers of two
    // the cut: tiles of R query rows (row r of a sequence and key head: token r / group, head r % group), their keys in `splits`
    // ranges of `chunk` (the last takes what is left). Narrow kernel: tiles_max of every sequence, tiles from tiles_max on are not
    // cut. 128-row tiles: tiles_max of all sequences together, counted through (kv_tile_of).
    int splits, chunk, tiles_max;
    float* part;         // [tile][key head][split]: R rows of 128 sums, then R maxima (of S), R denominators, R factors f (KA_ROW words a row)
    int few_max;         // both kernels run: sequences of up to so many query rows belong to the narrow one (0: one kernel has all)
};

// Weights are formed as 2^((S - m) f + 14), m the largest S of the row so far: small ones keep their bits in fp16. The difference comes first:
// it is never above 0 and exact where weights count, so that no weight passes 2^14 and the largest is 2^14 however large the
// scores S f are. (As 2^(S f - (m f - 14)), rounded at m f, weights overflowed or all vanished from scores of 2^25 on.)
constexpr float KA_P = 14.f;
constexpr int KA_ROW = KV_D + 3;  // words of a row's partial result

// what is visible: positions 0 .. kv_visible - 1 to token t of a sequence (as far as the table goes)
__device__ __forceinline__ int kv_visible(const KvRows& b, const KvSeq& s, int t) {
    const int64_t cap = b.table_ld << b.page_log;
    return int(min(int64_t(max(s.len - s.nq + t + 1, 0)), cap));
}

// Dimension d of a row whose sum came out as NaN though its scores are finite: there are values that are not. Every weight is above 0, so
// the sum of these values alone is the result: the infinity among them, NaN beside one of the other sign or a NaN. (In the products 0 *
// infinity spoils it: the lower half of a weight is often 0. To search every tile for infinities would cost every call.)
__device__ __forceinline__ float kv_not_finite(const KvAttnArgs& a, int s, int j, int vis, int d) {
    const int64_t plane = int64_t(a.rows.page) * KV_D;
    float sum = 0.f;
#pragma unroll 1
    for (int key0 = 0; key0 < vis && sum == sum; key0 += 16) {  // (a page holds 16 positions at least)
        const int pg = kv_page(a.rows, s, key0);
        if (pg < 0) continue;
        const __half* v = a.pool + ((int64_t(pg) * 2 + 1) * a.HKV + j) * a.planes * plane + (key0 & (a.rows.page - 1)) * KV_D + d;
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
            if (key0 + i >= vis) continue;
            float x = __half2float(v[i * KV_D]);
            if (a.planes == 2) x += __half2float(v[plane + i * KV_D]);
            if (!(fabsf(x) < INFINITY)) sum += x;
        }
    }
    return sum == 0.f ? NAN : sum;
}

// The u-th 128-row tile of a batch: its sequence and its number there; false when there are fewer. A whole warp calls it with the same u.
__device__ __forceinline__ bool kv_tile_of(const KvAttnArgs& a, int u, int* s, int* i) {
    if (a.rows.n_seq == 1) {
        *s = 0;
        *i = u;
        const KvSeq q = kv_seq(a.rows, 0);
        return int64_t(u) * 128 < int64_t(q.nq) * a.group;
    }
    const int lane = threadIdx.x & 31;
    for (int s0 = 0; s0 < a.rows.n_seq; s0 += 32) {
        int tiles = 0;
        if (s0 + lane < a.rows.n_seq) {
            const int lo = min(max(a.rows.q_start[s0 + lane], 0), a.rows.n_tok);
            const int rows = (min(max(a.rows.q_start[s0 + lane + 1], lo), a.rows.n_tok) - lo) * a.group;
            tiles = rows > a.few_max ? (rows + 127) / 128 : 0;
        }
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned here = __ballot_sync(0xffffffffu, upto > u);
        if (here) {
            const int l = __ffs(int(here)) - 1;
            *s = s0 + l;
            *i = u - __shfl_sync(0xffffffffu, upto - tiles, l);
            return true;
        }
        u -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cp16z(uint32_t dst, const void* src, bool on) {  // zeros when off
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

// (x, y) -> two packed fp16 and what they leave, packed; a remainder of an infinity is 0
__device__ __forceinline__ void half_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(isinf(f.x) ? 0.f : x - f.x, isinf(f.y) ? 0.f : y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
// the same for finite values
__device__ __forceinline__ void half_pair_finite(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Power of two 2^k that brings a row of queries with largest magnitude m into [2^14, 2^15), with the sign of the scale, and what undoes it in
// the scale. f is kept from 0 and infinity, which would make NaN of the -infinity of masked scores and of S - m = 0: S is below
// 2^39, so that below 1e-37 all scores are 0, and at the largest fp32 number all but the largest weigh nothing.
struct RowScale {
    Pow2 up;
    float f;  // |scale2| * 2^-k
};
__device__ __forceinline__ RowScale row_scale(float m, float scale2) {
    const int e = int((__float_as_uint(m) >> 23) & 255u);
    const int k = m > 0.f && e < 255 ? 14 - (max(e, 1) - 127) : 0;
    RowScale r{make_pow2(k), 0.f};
    const Pow2 down = make_pow2(-k);
    r.f = fminf(fmaxf(fabsf(scale2) * down.s1 * down.s2, 1e-37f), 3.4028235e38f);
    if (scale2 < 0.f) r.up.s1 = -r.up.s1;
    return r;
}

// Most positions of a sequence that the plans count with: what the caller expects, as far as the table goes (2^30 at most)
inline int kv_most(const Kv* kv, const elb_kv_batch* b) { return int(std::max<int64_t>(1, std::min(int64_t(b->max_len), b->table_ld * kv->page))); }

int kv_attn_few_prepare();
int kv_attn_tile_prepare();
int kv_attn_few_launch(const Kv* kv, KvAttnArgs a, const elb_kv_batch* b, cudaStream_t s);
size_t kv_attn_few_work(const Kv* kv, const elb_kv_batch* b, int n_head, int few_max);
// rows whose keys were cut: `tiles` tiles of `rows` (8, 16 or 128) query rows
int kv_attn_join(const KvAttnArgs& a, int rows, int64_t tiles, cudaStream_t s);
int kv_attn_tile_launch(const Kv* kv, int layer, KvAttnArgs a, const elb_kv_batch* b, cudaStream_t s);
size_t kv_attn_tile_work(const Kv* kv, const elb_kv_batch* b, int n_head, int few_max);

}  // namespace elb
