// Attention over a paged cache for few query rows per key head: single tokens of many sequences, or of one behind a long context
// (up to 16 rows = tokens x query heads of a key head; more are taken 16 at a time).
//
// Bound by memory: the keys and values are read once for all query heads of a key head, everything else is small. A
// CTA of four warps takes a range of the keys; a warp walks every fourth step of 16 keys on its own, with its own running
// maximum and sum (in fp32), its next steps on their way by cp.async into its own ring, and meets the others once at
// the end. A step is S^T = K q^T and O^T += V^T P^T on mma.sync m16n8k16: the keys and values are the 16-row operand, 8
// query rows the narrow one, so that the one to eight rows of a decode step waste nothing. (The tensor pipe is a fifth busy: tcgen05 with
// its 128 rows would leave 120 of them empty.) 64 tokens behind 100-8000 keys, 32 heads on 8, F16: 193 us, 6.3 TB/s; one behind
// 100003 keys, pairs: 131 us, 6.3 TB/s; one behind 41 keys 4.4 us.
//
// fp32 accuracy from fp16 operands: a query row is scaled by a power of two and held as hi + lo (22 bits), so are the
// weights; keys and values are what the cache holds, one fp16 or a pair. Products hi hi, hi lo, lo hi are exact, lo lo
// (2^-22) is left out. The tensor core adds with truncation: hi hi of a score is two chains of 4 MMAs, the small products one of 8 (of 16 with
// pairs, 2^-11 of the score together), a step's O^T one of 2 or 3 that starts from zero; what a chain ends in joins fp32 sums with rounding.
#include <algorithm>

#include "kv_attn.cuh"

namespace elb {

namespace {

constexpr int KF_WARPS = 4, KF_THREADS = 32 * KF_WARPS, KF_KEYS = 16;
constexpr int KF_LD = KV_D + 4;  // floats per row when the warps meet: no bank conflicts between rows

template <int PL, int NT> struct FewShape {
    static constexpr int ROWS = 8 * NT;
    static constexpr int STAGES = 3;
    static constexpr int TILE = KF_KEYS * KV_D * 2;  // bytes of 16 keys, one plane
    static constexpr int STAGE = 2 * PL * TILE;
    static constexpr int SMEM = KF_WARPS * STAGES * STAGE;
    static_assert(SMEM >= KF_WARPS * ROWS * (KF_LD + 4) * 4, "the warps' results take the place of the rings");
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t mtrans(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int PL, int NT>
__global__ void __launch_bounds__(KF_THREADS) k_kv_attn_few(const KvAttnArgs a) {
    using S = FewShape<PL, NT>;
    extern __shared__ __align__(128) uint8_t few_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    // block -> (sequence, key head, first tile, split), splits fastest
    int64_t x = blockIdx.x;
    const int c = int(x % a.splits);
    x /= a.splits;
    const int j = int(x % a.HKV);
    x /= a.HKV;
    const int i0 = int(x % a.tiles_max), s = int(x / a.tiles_max);
    const KvSeq sq = kv_seq(a.rows, s);
    const int nrows = sq.nq * a.group;
    if (a.few_max && nrows > a.few_max) return;
    const int64_t plane = int64_t(a.rows.page) * KV_D, head = PL * plane;
    const uint32_t ring = uint32_t(__cvta_generic_to_shared(few_smem)) + uint32_t(warp) * (S::STAGES * S::STAGE);

    for (int i = i0; i * S::ROWS < nrows; i += a.tiles_max) {
        const bool cut = a.splits > 1 && i < a.tiles_max;
        if (!cut && c) break;  // (the tiles that are not cut are those from tiles_max on)
        const int tok_last = min(((i + 1) * S::ROWS - 1) / a.group, sq.nq - 1);
        const int vis = kv_visible(a.rows, sq, tok_last), vis_min = kv_visible(a.rows, sq, i * S::ROWS / a.group);
        const int kb = cut ? c * a.chunk : 0, ke = cut && c < a.splits - 1 ? min(vis, kb + a.chunk) : vis;
        if (c && kb >= ke) continue;  // nothing here; the join does not look at it
        const int first = kb / KF_KEYS + warp, steps = (ke + KF_KEYS - 1) / KF_KEYS;
        const int mine = first < steps ? (steps - first + KF_WARPS - 1) / KF_WARPS : 0;

        int pages = -1;  // lane l: page of the warp's step number l, 32 + l, ...
        auto issue = [&](int n) {
            if ((n & 31) == 0) pages = n + lane < mine ? kv_page(a.rows, s, (first + KF_WARPS * (n + lane)) * KF_KEYS) : -1;
            const int pg = __shfl_sync(0xffffffffu, pages, n & 31);
            if (n < mine) {
                const int key0 = (first + KF_WARPS * n) * KF_KEYS;
                const __half* base = a.pool + (int64_t(max(pg, 0)) * 2 * a.HKV + j) * head + (key0 & (a.rows.page - 1)) * KV_D;
                const uint32_t st = ring + uint32_t(n % S::STAGES) * S::STAGE;
#pragma unroll
                for (int q = 0; q < S::TILE / 512; ++q) {
                    const int key = q * 2 + (lane >> 4), ch = lane & 15;
                    const bool on = pg >= 0 && key0 + key < vis;  // behind the last key: zeros, whatever lies there
                    const uint32_t d = st + uint32_t(key * 256 + ((ch ^ (key & 7)) << 4));
                    const __half* src = base + key * KV_D + ch * 8;
#pragma unroll
                    for (int pl = 0; pl < PL; ++pl) {
                        cp16z(d + pl * S::TILE, src + pl * plane, on);
                        cp16z(d + (PL + pl) * S::TILE, src + a.HKV * head + pl * plane, on);
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int n = 0; n < S::STAGES - 1; ++n) issue(n);

        // queries: lane (g, t) holds, of row g of each group of 8, the values 16 ks + 2 t, + 1, + 8, + 9 as hi and lo
        uint32_t qh[NT][8][2], ql[NT][8][2];
        float f[NT][2];     // factors of rows 2 t, 2 t + 1
        int see[NT][2];     // their visible keys
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = i * S::ROWS + nt * 8 + g;
            const float* src = a.q + (sq.row0 + r / a.group) * a.ldq + (j * a.group + r % a.group) * KV_D + 2 * t;
            float2 v[8][2];
            float m = 0.f;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    v[ks][b] = r < nrows ? *reinterpret_cast<const float2*>(src + 16 * ks + 8 * b) : make_float2(0.f, 0.f);
                    m = fmaxf(m, fmaxf(fabsf(v[ks][b].x), fabsf(v[ks][b].y)));
                }
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const RowScale rs = row_scale(m, a.scale2);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int b = 0; b < 2; ++b) half_pair(v[ks][b].x * rs.up.s1 * rs.up.s2, v[ks][b].y * rs.up.s1 * rs.up.s2, qh[nt][ks][b], ql[nt][ks][b]);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                f[nt][b] = __shfl_sync(0xffffffffu, rs.f, (2 * t + b) * 4);
                const int row = i * S::ROWS + nt * 8 + 2 * t + b;
                see[nt][b] = row < nrows ? kv_visible(a.rows, sq, row / a.group) : vis;
            }
        }

        float O[NT][8][4] = {}, m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int b = 0; b < 2; ++b) { m[nt][b] = -INFINITY; l[nt][b] = 0.f; }

        const int k_row = (lane & 15), k_chunk = lane >> 4;                       // K: rows 0-15, chunks 2 ks and 2 ks + 1
        const int v_row = (lane & 7) + ((lane >> 4) << 3), v_chunk = (lane >> 3) & 1;  // V transposed: chunks first, then rows 8-15
#pragma unroll 1
        for (int n = 0; n < mine; ++n) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
            __syncwarp();  // every lane's copies are there, and every lane is done with the stage that the next copies go to
            issue(n + S::STAGES - 1);
            const uint32_t st = ring + uint32_t(n % S::STAGES) * S::STAGE;
            const int key0 = (first + KF_WARPS * n) * KF_KEYS;
            float sh[NT][2][4] = {}, sx[NT][4] = {};
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                uint32_t kf[4], kl[4];
                const uint32_t ad = st + uint32_t(k_row * 256 + (((2 * ks + k_chunk) ^ (k_row & 7)) << 4));
                ldsm4(kf, ad);
                if (PL == 2) ldsm4(kl, ad + S::TILE);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16(sx[nt], kf, ql[nt][ks][0], ql[nt][ks][1]);
                    if (PL == 2) mma16(sx[nt], kl, qh[nt][ks][0], qh[nt][ks][1]);
                    mma16(sh[nt][ks & 1], kf, qh[nt][ks][0], qh[nt][ks][1]);
                }
            }
            uint32_t ph[NT][2], pl[NT][2];
            float p[NT][4], corr[NT][2];
            const bool edge = key0 + KF_KEYS > vis_min;  // some row does not see all of these keys
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {  // row 2 t + b: keys g and g + 8
                    float x0 = sh[nt][0][b] + sh[nt][1][b] + sx[nt][b];
                    float x1 = sh[nt][0][b + 2] + sh[nt][1][b + 2] + sx[nt][b + 2];
                    if (edge) {
                        if (key0 + g >= see[nt][b]) x0 = -INFINITY;
                        if (key0 + g + 8 >= see[nt][b]) x1 = -INFINITY;
                    }
                    float mx = fmaxf(x0, x1);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    mx = fmaxf(mx, m[nt][b]);
                    corr[nt][b] = mx == -INFINITY ? 1.f : ex2((m[nt][b] - mx) * f[nt][b]);
                    m[nt][b] = mx;
                    const float base = mx == -INFINITY ? 0.f : mx;
                    p[nt][b] = ex2(fmaf(x0 - base, f[nt][b], KA_P));
                    p[nt][b + 2] = ex2(fmaf(x1 - base, f[nt][b], KA_P));
                    l[nt][b] = l[nt][b] * corr[nt][b] + (p[nt][b] + p[nt][b + 2]);
                }
                half_pair_finite(p[nt][0], p[nt][1], ph[nt][0], pl[nt][0]);
                half_pair_finite(p[nt][2], p[nt][3], ph[nt][1], pl[nt][1]);
#pragma unroll
                for (int b = 0; b < 2; ++b) { ph[nt][b] = mtrans(ph[nt][b]); pl[nt][b] = mtrans(pl[nt][b]); }
            }
            bool odd = false;
            if (edge && vis_min < vis) {  // 0 * infinity must not reach a row that does not see the value
                uint32_t any = 0;
                const uint4* vv = reinterpret_cast<const uint4*>(few_smem + (st - uint32_t(__cvta_generic_to_shared(few_smem))) + PL * S::TILE);
                for (int w = lane; w < PL * S::TILE / 16; w += 32) {
                    const uint4 u = vv[w];
                    for (uint32_t h : {u.x, u.y, u.z, u.w}) any |= uint32_t((h & 0x7c00u) == 0x7c00u) | uint32_t((h & 0x7c000000u) == 0x7c000000u);
                }
                odd = __any_sync(0xffffffffu, any != 0);
            }
            if (!odd) {
#pragma unroll
                for (int mt = 0; mt < 8; ++mt) {
                    uint32_t vf[4], vl[4];
                    const uint32_t ad = st + uint32_t(PL * S::TILE + v_row * 256 + (((2 * mt + v_chunk) ^ (v_row & 7)) << 4));
                    ldsm4t(vf, ad);
                    if (PL == 2) ldsm4t(vl, ad + S::TILE);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float d[4] = {};
                        if (PL == 2) mma16(d, vl, ph[nt][0], ph[nt][1]);
                        mma16(d, vf, pl[nt][0], pl[nt][1]);
                        mma16(d, vf, ph[nt][0], ph[nt][1]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) O[nt][mt][e] = O[nt][mt][e] * corr[nt][e & 1] + d[e];
                    }
                }
            } else {  // key by key, for the rows that see it
                const __half* vv = reinterpret_cast<const __half*>(few_smem + (st - uint32_t(__cvta_generic_to_shared(few_smem))) + PL * S::TILE);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int mt = 0; mt < 8; ++mt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) O[nt][mt][e] *= corr[nt][e & 1];
#pragma unroll 1
                    for (int key = 0; key < KF_KEYS; ++key) {
                        const int from = (key & 7) * 4 + t;
                        float w[2];
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const float lo8 = __shfl_sync(0xffffffffu, p[nt][b], from), hi8 = __shfl_sync(0xffffffffu, p[nt][b + 2], from);
                            w[b] = key < 8 ? lo8 : hi8;
                        }
#pragma unroll
                        for (int mt = 0; mt < 8; ++mt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int d = mt * 16 + g + (e >> 1) * 8;
                                const int at = key * KV_D + (((d >> 3) ^ (key & 7)) << 3) + (d & 7);
                                float v = __half2float(vv[at]);
                                if (PL == 2) v += __half2float(vv[S::TILE / 2 + at]);
                                if (key0 + key < see[nt][e & 1]) O[nt][mt][e] += w[e & 1] * v;
                            }
                    }
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // the rings are free on every warp
        float* sO = reinterpret_cast<float*>(few_smem);  // [warp][row][KF_LD], then [warp][row] (m, l, f)
        float4* sml = reinterpret_cast<float4*>(sO + KF_WARPS * S::ROWS * KF_LD);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                float v = l[nt][b];
                v += __shfl_xor_sync(0xffffffffu, v, 4);
                v += __shfl_xor_sync(0xffffffffu, v, 8);
                v += __shfl_xor_sync(0xffffffffu, v, 16);
                if (g == 0) sml[warp * S::ROWS + nt * 8 + 2 * t + b] = make_float4(m[nt][b], v, f[nt][b], 0.f);
            }
            float* dst = sO + (warp * S::ROWS + nt * 8 + 2 * t) * KF_LD + g;
#pragma unroll
            for (int mt = 0; mt < 8; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) dst[(e & 1) * KF_LD + mt * 16 + (e >> 1) * 8] = O[nt][mt][e];
        }
        __syncthreads();
        if (NT == 2) {  // what each warp's sums count, once for all 128 dimensions (four tokens behind 300 keys 11.9 -> 11.3 us; 8 rows lose by the wait)
            if (tid < KF_WARPS * S::ROWS) {
                const int r = tid % S::ROWS;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < KF_WARPS; ++w) M = fmaxf(M, sml[w * S::ROWS + r].x);
                sml[tid].w = M == -INFINITY ? 1.f : ex2((sml[tid].x - M) * sml[tid].z);
            }
            __syncthreads();
        }
        const bool final_here = !cut || vis <= a.chunk;
        const int64_t slot = ((int64_t(s) * a.tiles_max + i) * a.HKV + j) * a.splits + c;
        float* part = a.part + slot * S::ROWS * KA_ROW;
        for (int r = 0; r < S::ROWS; ++r) {
            const int row = i * S::ROWS + r;
            if (row >= nrows) break;
            float M = -INFINITY, den = 0.f, num = 0.f;
#pragma unroll
            for (int w = 0; w < KF_WARPS; ++w) M = fmaxf(M, sml[w * S::ROWS + r].x);
#pragma unroll
            for (int w = 0; w < KF_WARPS; ++w) {
                const float4 ml = sml[w * S::ROWS + r];
                const float k = NT == 2 ? ml.w : M == -INFINITY ? 1.f : ex2((ml.x - M) * ml.z);
                den += k * ml.y;
                num += k * sO[(w * S::ROWS + r) * KF_LD + tid];
            }
            if (final_here) {
                float y = den == 0.f ? 0.f : num / den;
                if (y != y && den > 0.f) y = kv_not_finite(a, s, j, kv_visible(a.rows, sq, row / a.group), tid);
                a.out[(sq.row0 + row / a.group) * a.ldo + (j * a.group + row % a.group) * KV_D + tid] = y;
            } else {
                part[r * KV_D + tid] = num;
                if (tid == 0) { part[S::ROWS * KV_D + r] = M; part[S::ROWS * (KV_D + 1) + r] = den; part[S::ROWS * (KV_D + 2) + r] = sml[r].z; }
            }
        }
        __syncthreads();  // before the rings fill again
    }
}

// Rows whose keys were cut: a warp per (sequence, tile, key head, row) adds the ranges' sums in their order.
template <int ROWS>
__global__ void __launch_bounds__(256) k_kv_attn_join(const KvAttnArgs a) {
    const int lane = threadIdx.x & 31;
    pdl_wait();
    int64_t x = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int r = int(x % ROWS);
    x /= ROWS;
    const int64_t slot = x * a.splits;
    const int j = int(x % a.HKV);
    x /= a.HKV;
    int i = 0, s = 0;
    if (ROWS == 128) {
        if (x >= a.tiles_max || !kv_tile_of(a, int(x), &s, &i)) return;
    } else {
        i = int(x % a.tiles_max);
        s = int(x / a.tiles_max);
        if (s >= a.rows.n_seq) return;
    }
    const KvSeq sq = kv_seq(a.rows, s);
    if (ROWS != 128 && a.few_max && sq.nq * a.group > a.few_max) return;
    const int row = i * ROWS + r;
    if (row >= sq.nq * a.group) return;
    const int vis = kv_visible(a.rows, sq, min(((i + 1) * ROWS - 1) / a.group, sq.nq - 1));
    if (vis <= a.chunk) return;
    const int n = min(a.splits, (vis + a.chunk - 1) / a.chunk);
    const float* part = a.part + slot * ROWS * KA_ROW;
    const float f = part[ROWS * (KV_D + 2) + r];
    float M = -INFINITY;
    for (int c = lane; c < n; c += 32) M = fmaxf(M, part[c * ROWS * KA_ROW + ROWS * KV_D + r]);
    M = warp_max(M);
    float den = 0.f;
    float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < n; ++c) {
        const float* p = part + int64_t(c) * ROWS * KA_ROW;
        const float k = M == -INFINITY ? 1.f : ex2((p[ROWS * KV_D + r] - M) * f);
        const float4 v = *reinterpret_cast<const float4*>(p + r * KV_D + lane * 4);
        den += k * p[ROWS * (KV_D + 1) + r];
        num.x += k * v.x; num.y += k * v.y; num.z += k * v.z; num.w += k * v.w;
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    float* out = a.out + (sq.row0 + row / a.group) * a.ldo + (j * a.group + row % a.group) * KV_D + lane * 4;
    const float4 y = make_float4(num.x * inv, num.y * inv, num.z * inv, num.w * inv);
    *reinterpret_cast<float4*>(out) = y;
    if (den > 0.f && !((y.x + y.y) + (y.z + y.w) < INFINITY))
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
            const float z = e == 0 ? y.x : e == 1 ? y.y : e == 2 ? y.z : y.w;
            if (z != z) out[e] = kv_not_finite(a, s, j, kv_visible(a.rows, sq, row / a.group), lane * 4 + e);
        }
}

struct FewPlan { int nt, tiles, splits, chunk; };

FewPlan few_plan(const Kv* kv, const elb_kv_batch* b, int n_head, int few_max) {
    FewPlan p{};
    const int group = n_head / kv->HKV;
    int64_t rows = int64_t(std::max(1, std::min(b->max_q, b->n_tok))) * group;
    if (few_max) rows = few_max;
    // (beside the other kernel: mostly single tokens, whose rows fill one group of 8 when the heads do)
    p.nt = rows > 8 && !(few_max && group <= 8) ? 2 : 1;
    p.tiles = int((rows + 8 * p.nt - 1) / (8 * p.nt));
    const int resident = kv->sm_count * (kv->planes == 1 ? 2 : 1);
    const int64_t base = int64_t(b->n_seq) * kv->HKV * p.tiles;
    const int len = kv_most(kv, b);
    // One sequence: one wave of equal ranges. Several: lengths differ, ranges short enough for four waves, so that the last ones even
    // out. For 12, 8, 4, 2 waves, us, F16: 64 single tokens at 100-8000 keys 198, 199, 201, 206; 64 at 100-4000 98, 96, 93, 95; 16 at
    // 100-20000 52, 47, 44, 45; 256 at 700 131, 131, 116, 116; 64 of 4 tokens 128, 118, 114, 112.
    int64_t want = b->n_seq == 1 ? std::max<int64_t>(1, resident / base) : std::max<int64_t>(1, (int64_t(resident) * 4 + base - 1) / base);
    want = std::min<int64_t>(want, (len + 255) / 256);
    p.chunk = int((len + want - 1) / want + 63) / 64 * 64;
    p.splits = (len + p.chunk - 1) / p.chunk;
    return p;
}

template <int PL, int NT> int few_run(const KvAttnArgs& a, int64_t blocks, cudaStream_t s) {
    using S = FewShape<PL, NT>;
    auto kernel = k_kv_attn_few<PL, NT>;
    kernel<<<unsigned(blocks * a.splits), KF_THREADS, S::SMEM, s>>>(a);
    ELB_CUDA(cudaGetLastError());
    return a.splits > 1 ? kv_attn_join(a, S::ROWS, blocks, s) : ELB_OK;
}

}  // namespace

int kv_attn_few_prepare() {
    ELB_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(k_kv_attn_few<1, 1>), FewShape<1, 1>::SMEM));
    ELB_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(k_kv_attn_few<1, 2>), FewShape<1, 2>::SMEM));
    ELB_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(k_kv_attn_few<2, 1>), FewShape<2, 1>::SMEM));
    return ensure_dyn_smem(reinterpret_cast<const void*>(k_kv_attn_few<2, 2>), FewShape<2, 2>::SMEM);
}

int kv_attn_join(const KvAttnArgs& a, int rows, int64_t tiles, cudaStream_t s) {
    const unsigned blocks = unsigned((tiles * rows + 7) / 8);
    if (rows == 8) k_kv_attn_join<8><<<blocks, 256, 0, s>>>(a);
    else if (rows == 16) k_kv_attn_join<16><<<blocks, 256, 0, s>>>(a);
    else k_kv_attn_join<128><<<blocks, 256, 0, s>>>(a);
    ELB_CUDA(cudaGetLastError());
    return ELB_OK;
}

size_t kv_attn_few_work(const Kv* kv, const elb_kv_batch* b, int n_head, int few_max) {
    const FewPlan p = few_plan(kv, b, n_head, few_max);
    if (p.splits == 1) return 0;
    return size_t(b->n_seq) * p.tiles * kv->HKV * p.splits * 8 * p.nt * KA_ROW * 4;
}

int kv_attn_few_launch(const Kv* kv, KvAttnArgs a, const elb_kv_batch* b, cudaStream_t s) {
    const FewPlan p = few_plan(kv, b, a.H, a.few_max);
    a.splits = p.splits; a.chunk = p.chunk; a.tiles_max = p.tiles;
    const int64_t blocks = int64_t(b->n_seq) * p.tiles * kv->HKV;
    if (blocks * p.splits > 0x7fffffff || blocks * 2 * p.nt > 0x7fffffff) return fail(ELB_ERR_UNSUPPORTED, "kv_attention: too many rows");
    if (kv->planes == 1) return p.nt == 1 ? few_run<1, 1>(a, blocks, s) : few_run<1, 2>(a, blocks, s);
    return p.nt == 1 ? few_run<2, 1>(a, blocks, s) : few_run<2, 2>(a, blocks, s);
}

}  // namespace elb
