// Attention of new tokens over a paged cache (elb_kv_attention_dev): head h of the row at position p of a sequence,
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q.k_j - m),  j = 0..p,  m = the largest score so far,
// one pass over the keys with the running maximum and sum (when m grows, what has been added is multiplied by
// exp(m_old - m_new)). A row without keys gives 0.
#include <cmath>

#include "kv.cuh"

namespace elb {

namespace {

struct AttnArgs {
    KvRows rows;
    const __half* pool;  // this layer
    const float* q;
    float* out;
    int64_t ldq, ldo;
    int H, HKV, planes;
    float scale;
};

// One warp per (row, query head), four values of the head per lane.
__global__ void __launch_bounds__(256) k_kv_attn_rows(const AttnArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t item = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int t = int(item / a.H), h = int(item % a.H), kh = h / (a.H / a.HKV);
    if (t >= a.rows.n_tok) return;
    int seq = -1;
    for (int s = lane; s < a.rows.n_seq; s += 32)
        if (a.rows.q_start[s] <= t && t < a.rows.q_start[s + 1]) seq = s;
    seq = __reduce_max_sync(0xffffffffu, seq);
    if (seq < 0) return;
    const KvSeq sq = kv_seq(a.rows, seq);
    const int pos = sq.len - sq.nq + t - sq.row0;
    const float4 q = *reinterpret_cast<const float4*>(a.q + t * a.ldq + h * KV_D + lane * 4);
    const int64_t plane = int64_t(a.rows.page) * KV_D, head = a.planes * plane;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto get = [&](const __half* p) {
        uint2 r = *reinterpret_cast<const uint2*>(p);
        float2 x = __half22float2(*reinterpret_cast<__half2*>(&r.x)), y = __half22float2(*reinterpret_cast<__half2*>(&r.y));
        if (a.planes == 2) {
            r = *reinterpret_cast<const uint2*>(p + plane);
            const float2 u = __half22float2(*reinterpret_cast<__half2*>(&r.x)), v = __half22float2(*reinterpret_cast<__half2*>(&r.y));
            x.x += u.x; x.y += u.y; y.x += v.x; y.y += v.y;
        }
        return make_float4(x.x, x.y, y.x, y.y);
    };
    for (int j = 0; j <= pos; ++j) {
        const int pg = kv_page(a.rows, seq, j);
        float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
        if (pg >= 0) {
            const __half* base = a.pool + (int64_t(pg) * 2 * a.HKV + kh) * head + int64_t(j & (a.rows.page - 1)) * KV_D + lane * 4;
            k = get(base);
            v = get(base + a.HKV * head);
        }
        const float x = warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w) * a.scale;
        const float m2 = fmaxf(m, x), c = m2 == -INFINITY ? 1.f : expf(m - m2), w = x == -INFINITY ? 0.f : expf(x - m2);
        m = m2;
        l = l * c + w;
        o.x *= c; o.y *= c; o.z *= c; o.w *= c;
        if (w != 0.f) {
            o.x += w * v.x; o.y += w * v.y; o.z += w * v.z; o.w += w * v.w;
        }
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
    *reinterpret_cast<float4*>(a.out + t * a.ldo + h * KV_D + lane * 4) = o;
}

}  // namespace

size_t kv_attention_work(const Kv* kv, const elb_kv_batch* b, int n_head) {
    if (!kv || !b || n_head <= 0 || n_head % kv->HKV) return 0;
    return 256;
}

int kv_attention_launch(const Kv* kv, int layer, const elb_kv_batch* b, const float* q, int64_t ldq, int n_head, float scale, float* out,
                        int64_t ldo, void* work, size_t work_bytes, cudaStream_t s) {
    ELB_TRY(kv_check_batch(kv, layer, b, "kv_attention"));
    if (n_head <= 0 || n_head % kv->HKV || n_head / kv->HKV > 64)
        return fail(ELB_ERR_INVALID, "kv_attention: query heads must be a multiple of the key heads, at most 64 times them");
    if (!std::isfinite(scale)) return fail(ELB_ERR_INVALID, "kv_attention: the scale must be finite");
    if (b->n_tok == 0 || b->n_seq == 0) return ELB_OK;
    if (!q || !out) return fail(ELB_ERR_INVALID, "kv_attention: null argument");
    if (ldq < int64_t(n_head) * KV_D || ldo < int64_t(n_head) * KV_D) return fail(ELB_ERR_INVALID, "kv_attention: a row stride is shorter than the row");
    if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 16 || ldq % 4 || ldo % 4)
        return fail(ELB_ERR_UNSUPPORTED, "kv_attention: rows must start on 16-byte boundaries");
    if (!work || work_bytes < kv_attention_work(kv, b, n_head)) return fail(ELB_ERR_INVALID, "kv_attention: the work buffer is too small");
    if (reinterpret_cast<uintptr_t>(work) % 256) return fail(ELB_ERR_INVALID, "kv_attention: the work buffer must start on a 256-byte boundary");
    DeviceScope on(kv->device);
    if (on.rc != ELB_OK) return on.rc;
    AttnArgs a{kv_rows(kv, b), kv->mem + int64_t(layer) * kv->layer_halves(), q, out, ldq, ldo, n_head, kv->HKV, kv->planes, scale};
    const int64_t blocks = (int64_t(b->n_tok) * n_head + 7) / 8;
    if (blocks > 0x7fffffff) return fail(ELB_ERR_UNSUPPORTED, "kv_attention: too many rows");
    k_kv_attn_rows<<<unsigned(blocks), 256, 0, s>>>(a);
    ELB_CUDA(cudaGetLastError());
    return ELB_OK;
}

}  // namespace elb
