// Paged cache of keys and values: the handle, and how its kernels find rows, positions and pages.
#pragma once

#include <cuda.h>

#include <vector>

#include "common.cuh"

namespace elb {

constexpr int KV_D = 128;  // head_dim

struct Rope {
    int device = 0, head_dim = 0, dim = 0, layout = 0;
    double* d_turns = nullptr;  // [dim/2] full turns per position, f_i / 2 pi
    float mscale = 1.f;
};

struct Kv {
    int device = 0, n_layer = 0, HKV = 0, page = 0, n_pages = 0, planes = 1, sm_count = 0;
    __half* mem = nullptr;
    bool owned = false;
    int *err = nullptr, *err_dev = nullptr;  // pinned word that a kernel raises when one of its bounded waits runs out, and its device address
    CUtensorMap map{};  // the pool as rows of 128 halves, box of 64 halves x min(page, 64) rows, 128-byte swizzle
    int64_t head_halves() const { return int64_t(planes) * page * KV_D; }         // keys or values of one head in a page
    int64_t page_halves() const { return 2 * HKV * head_halves(); }              // one page of one layer
    int64_t layer_halves() const { return int64_t(n_pages) * page_halves(); }
};

// The batch as kernels read it. Nothing on the device is trusted to be in range.
struct KvRows {
    const int *q_start, *len, *table;
    int64_t table_ld;
    int n_seq, n_tok;
    int page, page_log, n_pages;
};

struct KvSeq {
    int row0, nq, len;  // first row, rows, positions (0 when negative; may exceed the table)
};
__device__ __forceinline__ KvSeq kv_seq(const KvRows& b, int s) {
    KvSeq q;
    q.row0 = min(max(b.q_start[s], 0), b.n_tok);
    q.nq = min(max(b.q_start[s + 1], q.row0), b.n_tok) - q.row0;
    q.len = max(b.len[s], 0);
    return q;
}
// page of position p of sequence s, or -1 when the table has none or it is outside the pool
__device__ __forceinline__ int kv_page(const KvRows& b, int s, int p) {
    const int i = p >> b.page_log;
    if (p < 0 || i >= b.table_ld) return -1;
    const int pg = b.table[s * b.table_ld + i];
    return unsigned(pg) < unsigned(b.n_pages) ? pg : -1;
}

inline KvRows kv_rows(const Kv* kv, const elb_kv_batch* b) {
    int log = 0;
    while ((1 << log) < kv->page) ++log;
    return KvRows{b->d_q_start, b->d_len, b->d_table, b->table_ld, b->n_seq, b->n_tok, kv->page, log, kv->n_pages};
}

// The handle's device for the length of a call; the caller's comes back at its end.
struct DeviceScope {
    int before = -1, rc = ELB_OK;
    explicit DeviceScope(int device) {
        if (cudaGetDevice(&before) != cudaSuccess || (before != device && cudaSetDevice(device) != cudaSuccess)) {
            rc = fail(ELB_ERR_CUDA, std::string("cannot use the handle's device: ") + cudaGetErrorString(cudaGetLastError()));
            before = -1;
        } else if (before == device) {
            before = -1;
        }
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// Do n rows of wx floats, ldx apart from x on, share memory with n rows of wy floats, ldy apart from y on? Columns of one buffer (equal
// strides) are told apart; with unequal strides ranges that interleave count as apart.
inline bool rows_meet(const float* x, int64_t ldx, int64_t wx, const float* y, int64_t ldy, int64_t wy, int64_t n) {
    using Wide = __int128;
    const Wide ux = Wide(reinterpret_cast<uintptr_t>(x)), uy = Wide(reinterpret_cast<uintptr_t>(y));
    if (ux + (Wide(n - 1) * ldx + wx) * 4 <= uy || uy + (Wide(n - 1) * ldy + wy) * 4 <= ux) return false;
    if (n == 1) return true;
    if (ldx != ldy) return false;
    const Wide row = Wide(ldx) * 4;
    Wide r = (uy - ux) % row;
    if (r < 0) r += row;
    const Wide k = (uy - ux - r) / row;  // row j of y starts r bytes behind the start of row k + j of x, row - r in front of the next one's
    return (r < wx * 4 && k < n && -k < n) || (row - r < wy * 4 && k + 1 < n && -k - 1 < n);
}

// rope.cu
int rope_frequencies(const elb_rope_config* c, std::vector<double>* freq, double* m);
int rope_create(int device, const elb_rope_config* c, Rope** out);
void rope_destroy(Rope* r);
int rope_launch(const Rope* r, const float* x, int64_t ldx, float* y, int64_t ldy, int64_t n, int heads, const int* pos, const float* norm,
                float eps, cudaStream_t s);
int kv_append_launch(Kv* kv, int layer, const elb_kv_batch* b, const Rope* rope, const float* k, int64_t ldk, const float* v, int64_t ldv,
                     const float* k_norm, float eps, const float* q, int64_t ldq, int n_head, const float* q_norm, float* q_out, int64_t ldqo,
                     cudaStream_t s);
// kv.cu
size_t kv_bytes(int n_layer, int n_head_kv, int head_dim, int page, int n_pages, int type);
int kv_create(int device, int n_layer, int n_head_kv, int head_dim, int page, int n_pages, int type, void* mem, Kv** out);
void kv_destroy(Kv* kv);
int kv_check_batch(const Kv* kv, int layer, const elb_kv_batch* b, const char* what);
int kv_reorder_launch(Kv* kv, int n, const int* parent, const int* len, const int* table, int64_t table_ld, const int* spare, int* len_out,
                      int* table_out, int* taken, cudaStream_t s);
// kv_attn.cu
size_t kv_attention_work(const Kv* kv, const elb_kv_batch* b, int n_head);
int kv_attention_launch(const Kv* kv, int layer, const elb_kv_batch* b, const float* q, int64_t ldq, int n_head, float scale, float* out,
                        int64_t ldo, void* work, size_t work_bytes, cudaStream_t s);
int kv_attention_prepare();  // on the current device: what a captured call must find in place
int kv_attention_check(const Kv* kv);  // did a kernel of an earlier call on this cache give up on a bounded wait?
int kv_attention_wait_expiry(const Kv* kv);
// beam.cu
size_t beam_select_work(int n_vocab, int n_group, int beams, int k);
int beam_select_launch(int device, const float* logits, int64_t ld, int n_vocab, int n_group, int beams, const double* scores,
                       const uint32_t* allowed, int64_t allowed_ld, int k, int* parent, int* token, double* score, void* work, size_t work_bytes,
                       cudaStream_t s);

}  // namespace elb
