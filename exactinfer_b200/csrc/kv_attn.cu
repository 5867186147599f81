// Attention of new tokens over a paged cache (elb_kv_attention_dev): head h of the row at position p of a sequence,
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q.k_j - m),  j = 0..p,  m = the largest score so far,
// one pass over the keys with the running maximum and sum (when m grows, what has been added is multiplied by
// exp(m_old - m_new)). A row without keys gives 0.
#include <algorithm>
#include <cmath>

#include "kv_attn.cuh"

namespace elb {

// Up to 16 query rows per key head go to the narrow kernel, more to the 128-row tiles. A batch that may hold many sequences of
// either kind (a server's step with a chunk of somebody's prompt in it) takes both, each for its sequences: 63 single tokens and a
// chunk of 512 rows behind 100-4000 keys 296 -> 160 us. few_max: 0 for one kernel, else the rows up to which a sequence is
// the narrow one's.
constexpr int FEW_ROWS = 16;
struct AttnWay { bool few, tile; int few_max; };
static AttnWay attn_way(const elb_kv_batch* b, int group) {
    const int64_t most = std::min(b->max_q, b->n_tok);
    if (most * group <= FEW_ROWS) return {true, false, 0};
    const bool both = b->n_seq >= 4 && 2 * int64_t(b->n_tok) < b->n_seq * most;
    return {both, true, both ? FEW_ROWS : 0};
}
static size_t up256(size_t x) { return (x + 255) / 256 * 256; }

int kv_attention_prepare() {
    ELB_TRY(kv_attn_few_prepare());
    return kv_attn_tile_prepare();
}

size_t kv_attention_work(const Kv* kv, const elb_kv_batch* b, int n_head) {
    if (!kv || !b || n_head <= 0 || n_head % kv->HKV || n_head / kv->HKV > 64) return 0;
    if (b->n_seq < 0 || b->n_seq > 65536 || b->n_tok < 0 || b->max_q < 0 || b->max_len < 0 || b->table_ld < 0 || b->table_ld > (int64_t(1) << 30) / kv->page) return 0;
    if (b->n_seq == 0 || b->n_tok == 0) return 256;  // (the call has nothing to do, and the plans below divide by the sequences)
    if (b->table_ld == 0) return 0;
    const AttnWay w = attn_way(b, n_head / kv->HKV);
    return std::max<size_t>(256, (w.few ? up256(kv_attn_few_work(kv, b, n_head, w.few_max)) : 0) + (w.tile ? kv_attn_tile_work(kv, b, n_head, w.few_max) : 0));
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
    if (rows_meet(q, ldq, int64_t(n_head) * KV_D, out, ldo, int64_t(n_head) * KV_D, b->n_tok)) return fail(ELB_ERR_INVALID, "kv_attention: the output must not overlap the queries");
    if (!work || work_bytes < kv_attention_work(kv, b, n_head)) return fail(ELB_ERR_INVALID, "kv_attention: the work buffer is too small");
    if (reinterpret_cast<uintptr_t>(work) % 256) return fail(ELB_ERR_INVALID, "kv_attention: the work buffer must start on a 256-byte boundary");
    DeviceScope on(kv->device);
    if (on.rc != ELB_OK) return on.rc;
    KvAttnArgs a{};
    a.rows = kv_rows(kv, b);
    a.pool = kv->mem + int64_t(layer) * kv->layer_halves();
    a.q = q; a.out = out; a.ldq = ldq; a.ldo = ldo;
    a.H = n_head; a.HKV = kv->HKV; a.group = n_head / kv->HKV; a.planes = kv->planes;
    a.scale2 = scale * 1.44269504088896340736f;
    const AttnWay w = attn_way(b, a.group);
    a.few_max = w.few_max;
    uint8_t* at = static_cast<uint8_t*>(work);
    ELB_TRY(kv_attention_check(kv));
    if (w.few) {
        a.part = reinterpret_cast<float*>(at);
        at += up256(kv_attn_few_work(kv, b, n_head, w.few_max));
        ELB_TRY(kv_attn_few_launch(kv, a, b, s));
    }
    if (!w.tile) return ELB_OK;
    a.part = reinterpret_cast<float*>(at);
    return kv_attn_tile_launch(kv, layer, a, b, s);
}

}  // namespace elb
