// The paged cache's handle, and the reordering of states after a beam search's selection (elb_kv_reorder_dev).
#include <cuda.h>

#include <algorithm>

#include <new>

#include "kv.cuh"

namespace elb {

namespace {

constexpr int KR_THREADS = 256, KR_MAXROWS = 4096, KR_CHUNK = 16384;  // KR_CHUNK: bytes of one piece of a page

// Row r goes on from row parent[r]. Its first child keeps a last page that is not full, every other child gets a copy in
// its spare page. The copies of all layers are cut into pieces of 16 KB and dealt out evenly over the blocks; every block
// works out the list of copies for itself (n words of shared memory: cheaper than a launch before this one). Bound by memory: bytes
// of the copied pages, read and written once (64 rows, 12 layers, 119 MB: 23 us, 5.2 TB/s).
__global__ void __launch_bounds__(KR_THREADS) k_kv_reorder(uint8_t* __restrict__ pool, int64_t layer_bytes, int64_t page_bytes, int n_layer,
                                                           int n_pages, int page, int n, const int* __restrict__ parent,
                                                           const int* __restrict__ len, const int* __restrict__ table, int64_t table_ld,
                                                           const int* __restrict__ spare, int* __restrict__ len_out,
                                                           int* __restrict__ table_out, int* __restrict__ taken) {
    extern __shared__ int sh[];
    int* first = sh;                    // [n] lowest child of each row
    int2* copy = reinterpret_cast<int2*>(sh + (n + 1) / 2 * 2);  // [n] (from page, to page)
    __shared__ int warp_count[KR_THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int r = tid; r < n; r += KR_THREADS) first[r] = n;
    __syncthreads();
    for (int r = tid; r < n; r += KR_THREADS) {
        const int p = parent[r];
        if (unsigned(p) < unsigned(n)) atomicMin(first + p, r);
    }
    __syncthreads();
    int copies = 0;  // the same in every thread and block
    for (int r0 = 0; r0 < n; r0 += KR_THREADS) {
        const int r = r0 + tid;
        bool on = false;
        int2 ft = make_int2(-1, -1);
        int keep_len = 0, last = 0;
        if (r < n) {
            const int p = parent[r];
            const bool live = unsigned(p) < unsigned(n);
            keep_len = live ? max(len[p], 0) : 0;
            last = keep_len / page;
            if (live && keep_len % page && first[p] != r && last < table_ld) {
                ft = make_int2(table[p * table_ld + last], spare[r]);
                on = unsigned(ft.x) < unsigned(n_pages) && unsigned(ft.y) < unsigned(n_pages);
            }
        }
        const unsigned vote = __ballot_sync(0xffffffffu, on);
        if (lane == 0) warp_count[warp] = __popc(vote);
        __syncthreads();
        int at = copies;
        for (int w = 0; w < KR_THREADS / 32; ++w) {
            if (w < warp) at += warp_count[w];
            copies += warp_count[w];
        }
        if (on) copy[at + __popc(vote & ((1u << lane) - 1u))] = ft;
        __syncthreads();
        if (r < n && r % gridDim.x == blockIdx.x) {  // (the rows' words are few: one thread each)
            taken[r] = on;
            len_out[r] = keep_len;
        }
    }
    // tables: a warp per row
    const int warps = int(gridDim.x) * (KR_THREADS / 32);
    for (int r = int(blockIdx.x) * (KR_THREADS / 32) + warp; r < n; r += warps) {
        const int p = parent[r];
        const bool live = unsigned(p) < unsigned(n);
        const int l = live ? max(len[p], 0) : 0, used = l / page + (l % page != 0);
        const bool second = live && l % page && first[p] != r;
        for (int64_t i = lane; i < table_ld; i += 32) {
            int v = -1;
            if (i < used) {
                v = table[p * table_ld + i];
                if (second && i == used - 1 && unsigned(v) < unsigned(n_pages)) v = spare[r];  // (one outside the pool: not the first child's page either)
            }
            table_out[r * table_ld + i] = v;
        }
    }
    const int64_t pieces = (page_bytes + KR_CHUNK - 1) / KR_CHUNK, work = int64_t(copies) * n_layer * pieces;
    for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
        const int64_t piece = w % pieces, rest = w / pieces;
        const int2 ft = copy[rest / n_layer];
        uint8_t* base = pool + (rest % n_layer) * layer_bytes;
        const uint4* src = reinterpret_cast<const uint4*>(base + ft.x * page_bytes + piece * KR_CHUNK);
        uint4* dst = reinterpret_cast<uint4*>(base + ft.y * page_bytes + piece * KR_CHUNK);
        const int words = int(min(int64_t(KR_CHUNK), page_bytes - piece * KR_CHUNK) / 16);
        uint4 v[KR_CHUNK / 16 / KR_THREADS];
#pragma unroll
        for (int j = 0; j < KR_CHUNK / 16 / KR_THREADS; ++j)
            if (tid + j * KR_THREADS < words) v[j] = __ldcg(src + tid + j * KR_THREADS);
#pragma unroll
        for (int j = 0; j < KR_CHUNK / 16 / KR_THREADS; ++j)
            if (tid + j * KR_THREADS < words) __stcg(dst + tid + j * KR_THREADS, v[j]);
    }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

bool page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128 || page == 256; }

}  // namespace

size_t kv_bytes(int n_layer, int n_head_kv, int head_dim, int page, int n_pages, int type) {
    if (n_layer <= 0 || n_layer > 4096 || n_head_kv <= 0 || n_head_kv > 4096 || n_pages <= 0 || !page_ok(page) || head_dim != KV_D ||
        (type != ELB_KV_F16 && type != ELB_KV_PAIR))
        return 0;
    const double rows = double(n_layer) * n_pages * 2 * n_head_kv * type * page;
    if (rows >= 2147483648.0) return 0;  // (row numbers are 32-bit coordinates of the tensor loads)
    return size_t(rows) * KV_D * 2;
}

int kv_create(int device, int n_layer, int n_head_kv, int head_dim, int page, int n_pages, int type, void* mem, Kv** out) {
    if (!out) return fail(ELB_ERR_INVALID, "kv_create: null argument");
    if (head_dim != KV_D) return fail(ELB_ERR_UNSUPPORTED, "kv_create: only head_dim = 128 is supported");
    if (!page_ok(page)) return fail(ELB_ERR_UNSUPPORTED, "kv_create: a page holds 16, 32, 64, 128 or 256 positions");
    if (type != ELB_KV_F16 && type != ELB_KV_PAIR) return fail(ELB_ERR_UNSUPPORTED, "kv_create: unknown type of values");
    if (n_layer <= 0 || n_head_kv <= 0 || n_pages <= 0) return fail(ELB_ERR_INVALID, "kv_create: layers, heads and pages must be positive");
    const size_t bytes = kv_bytes(n_layer, n_head_kv, head_dim, page, n_pages, type);
    if (!bytes) return fail(ELB_ERR_UNSUPPORTED, "kv_create: the pool is too large (2^31 rows of 128 values at most)");
    if (reinterpret_cast<uintptr_t>(mem) % 128) return fail(ELB_ERR_INVALID, "kv_create: the pool's memory must start on a 128-byte boundary");
    DeviceScope on(device);
    if (on.rc != ELB_OK) return on.rc;
    DeviceInfo di;
    ELB_TRY(device_info(device, &di));
    void* fp = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fp, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
        return fail(ELB_ERR_CUDA, "kv_create: cuTensorMapEncodeTiled is not available");
    ELB_TRY(kv_attention_prepare());
    ELB_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(k_kv_reorder), KR_MAXROWS * 12));
    auto* kv = new (std::nothrow) Kv;
    if (!kv) return fail(ELB_ERR_MEMORY, "kv_create: out of memory");
    kv->device = device; kv->n_layer = n_layer; kv->HKV = n_head_kv; kv->page = page; kv->n_pages = n_pages; kv->planes = type;
    kv->sm_count = di.sm_count;
    kv->mem = static_cast<__half*>(mem);
    if (cudaHostAlloc(&kv->err, sizeof(int), cudaHostAllocMapped) != cudaSuccess || cudaHostGetDevicePointer(&kv->err_dev, kv->err, 0) != cudaSuccess) {
        cudaGetLastError();
        if (kv->err) cudaFreeHost(kv->err);
        delete kv;
        return fail(ELB_ERR_MEMORY, "kv_create: no error word");
    }
    *kv->err = 0;
    if (!mem) {
        if (device_malloc(&kv->mem, bytes) != cudaSuccess) {
            cudaFreeHost(kv->err);
            delete kv;
            return fail(ELB_ERR_MEMORY, "kv_create: out of device memory");
        }
        kv->owned = true;
        cudaError_t e = cudaMemset(kv->mem, 0, bytes);  // (returns before it is done, and a caller's stream need not wait for the default one)
        if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
        if (e != cudaSuccess) {
            kv_destroy(kv);
            return fail(ELB_ERR_CUDA, std::string("kv_create: ") + cudaGetErrorString(e));
        }
    }
    const cuuint64_t dims[2] = {KV_D, bytes / (KV_D * 2)}, strides[1] = {KV_D * 2};
    const cuuint32_t box[2] = {64, cuuint32_t(std::min(page, 64))}, es[2] = {1, 1};
    const CUresult r = reinterpret_cast<EncodeFn>(fp)(&kv->map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, kv->mem, dims, strides, box, es,
                                                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        kv_destroy(kv);
        return fail(ELB_ERR_CUDA, "kv_create: tensor map encoding failed");
    }
    *out = kv;
    return ELB_OK;
}

void kv_destroy(Kv* kv) {
    if (!kv) return;
    DeviceScope on(kv->device);
    if (kv->owned) cudaFree(kv->mem);
    else cudaDeviceSynchronize();
    cudaFreeHost(kv->err);
    delete kv;
}

int kv_check_batch(const Kv* kv, int layer, const elb_kv_batch* b, const char* what) {
    if (!kv || !b) return fail(ELB_ERR_INVALID, std::string(what) + ": null argument");
    if (layer < 0 || layer >= kv->n_layer) return fail(ELB_ERR_RANGE, std::string(what) + ": layer out of range");
    if (b->n_seq < 0 || b->n_tok < 0 || b->max_q < 0 || b->max_len < 0) return fail(ELB_ERR_INVALID, std::string(what) + ": negative count");
    if (b->n_seq > 65536) return fail(ELB_ERR_UNSUPPORTED, std::string(what) + ": more than 65536 sequences");
    if (b->n_seq > 0 && b->n_tok > 0 && (!b->d_q_start || !b->d_len || !b->d_table)) return fail(ELB_ERR_INVALID, std::string(what) + ": null argument");
    if (b->table_ld < 0 || (b->n_seq > 0 && b->table_ld == 0)) return fail(ELB_ERR_INVALID, std::string(what) + ": a page table needs a positive row stride");
    if (b->table_ld > (int64_t(1) << 30) / kv->page) return fail(ELB_ERR_UNSUPPORTED, std::string(what) + ": tables for more than 2^30 positions");  // (a pool has fewer)
    return ELB_OK;
}

int kv_reorder_launch(Kv* kv, int n, const int* parent, const int* len, const int* table, int64_t table_ld, const int* spare, int* len_out,
                      int* table_out, int* taken, cudaStream_t s) {
    if (!kv) return fail(ELB_ERR_INVALID, "kv_reorder: null argument");
    if (n < 0 || table_ld < 0) return fail(ELB_ERR_INVALID, "kv_reorder: negative count");
    if (n > KR_MAXROWS) return fail(ELB_ERR_UNSUPPORTED, "kv_reorder: more than 4096 rows");
    if (n == 0) return ELB_OK;
    if (!parent || !len || !table || !spare || !len_out || !table_out || !taken || table_ld == 0) return fail(ELB_ERR_INVALID, "kv_reorder: null argument");
    auto apart = [](const void* a, size_t na, const void* b, size_t nb) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
        return x + na <= y || y + nb <= x;
    };
    const size_t row = size_t(n) * 4, tab = row * size_t(table_ld);
    const void* in[4] = {parent, len, table, spare};
    const void* out[3] = {len_out, table_out, taken};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 3; ++j)
            if (!apart(in[i], i == 2 ? tab : row, out[j], j == 1 ? tab : row)) return fail(ELB_ERR_INVALID, "kv_reorder: outputs must not overlap inputs");
    DeviceScope on(kv->device);
    if (on.rc != ELB_OK) return on.rc;
    const size_t smem = size_t((n + 1) / 2 * 2) * 4 + size_t(n) * 8;
    const int64_t page_bytes = kv->page_halves() * 2, most = (int64_t(n) * kv->n_layer * page_bytes + KR_CHUNK - 1) / KR_CHUNK;
    const int grid = int(std::min<int64_t>(std::max<int64_t>(most, 1), int64_t(kv->sm_count) * 4));
    k_kv_reorder<<<grid, KR_THREADS, smem, s>>>(reinterpret_cast<uint8_t*>(kv->mem), kv->layer_halves() * 2, page_bytes, kv->n_layer, kv->n_pages,
                                                kv->page, n, parent, len, table, table_ld, spare, len_out, table_out, taken);
    ELB_CUDA(cudaGetLastError());
    return ELB_OK;
}

}  // namespace elb
