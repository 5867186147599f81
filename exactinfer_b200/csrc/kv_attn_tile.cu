// Attention over a paged cache for many query rows per key head (prompts, chunks of a prompt, turns of a conversation), on the
// 5th-generation tensor cores.
//
// A CTA takes 128 query rows of one sequence and key head (tokens x the query heads that share the key head) and walks the keys
// that they see, 128 at a time: S = Q K^T, weights 2^((S - m) f + 14), O += P V. fp32 accuracy from fp16 operands as in
// kv_attn_few.cu: a query row is scaled by a power of two and held as hi + lo (22 bits), the weights as well, keys and
// values are one fp16 or a pair as the cache holds them; lo lo is left out, so that a product costs 2 MMAs (F16 cache) or 3 (pairs).
// The tensor core adds with truncation: the small products of a step go first, hi hi (8 links for S, 4 for O) last, and
// a step's O starts from zero and joins the running sum in registers, in fp32 with rounding, behind the factor
// 2^(m_old - m_new) - tensor memory never needs rescaling.
//
// Two teams of four warps work on alternate key tiles, a thread per query row (= TMEM lane), each with its own running
// maximum, denominator and 128 sums, joined once at the end: while one team forms its weights, the tensor core
// multiplies for the other. Warp 8 brings keys and values by TMA, page by page, into a ring of 128-key tiles in the order of their
// use; warps 9 and 10 issue the MMAs, one per team; warp 11 searches the values of edge tiles. TMEM: Q hi | lo (128 columns, the A
// operand of S: read from there, the shared memory has only K to deliver), per team S (128 columns, overwritten by the weights
// hi | lo, the A operand of O) and one O (128): a team takes it into its registers while the tensor core forms the next S. V lies
// [key][dimension] as in the page and is a B operand with N along the rows.
// A tile's 128 keys take 2048 (F16) or 3 * 1024 (pairs) clocks of the tensor pipe. (64-key tiles: an MMA with N = 64 took 51
// clocks instead of 32, and the whole 1860 a tile.) What bounds it is the chain S, weights, O, sums of a tile with one O: the
// tensor pipe is 54 to 59 % busy. 4096 causal rows, 32 query heads on 8: F16 257 us (535 TFLOP/s of useful products, 1070 of both
// halves), pairs 348 us (335 to 365 with the clock under the power cap). (Four teams' warps with half a row a thread: 277 us.)
//
// Behind the last visible key the weights are 0, but 0 * NaN is not: the PV product stops at the last 16 keys, and the rows of
// V behind the last key are emptied in shared memory. In the few tiles that only some rows see, V is searched for infinities and
// NaN; where there are any, the tile's product is done by the threads, key by key, for the rows that see it. Infinite values that a row does
// see are left to its end: where a result is NaN, they are added up by themselves (kv_not_finite).
#include <algorithm>

#include "kv_attn.cuh"

namespace elb {

namespace {

constexpr int KT_ROWS = 128, KT_KEYS = 128, KT_THREADS = 384, KT_MAXEDGE = 4;
constexpr unsigned KT_SPIN = 1u << 21;
constexpr int KT_LD = KV_D + 4;  // floats per row when the teams meet

template <int PL> struct TileShape {
    static constexpr int HALF = KT_KEYS * 128;           // 64 of the 128 values of every key
    static constexpr int PLANE = 2 * HALF;               // one plane
    static constexpr int SLOT = PL * PLANE;              // keys or values of a tile
    static constexpr int SLOTS = 6 / PL;
    static constexpr int RING = SLOTS * SLOT;
    static constexpr int SMEM = RING + 4096 + 1024;
    static constexpr int Q_STAGE = RING - KT_ROWS * KT_LD * 4;  // the queries pass through the end of the ring
    static_assert(RING >= 2 * KT_ROWS * KT_LD * 4, "the teams' sums take the place of the ring");
};

struct TileBars {
    uint64_t full[6], empty[6], s_full[2], pv_ready[2], o_full[2], q_full, go[KT_MAXEDGE], edge[KT_MAXEDGE];
    uint32_t tmem;
    int odd[KT_MAXEDGE];  // edge tile k has infinities or NaN among its values
    int fail;
};

__device__ __forceinline__ uint32_t su32(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint64_t* b, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory"); }
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(su32(b)), "r"(parity) : "memory");
    return done != 0;
}
// bounded: false when it ran out, or when another warp's wait has
template <unsigned SPIN = KT_SPIN> __device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity, TileBars* bars) {
    for (unsigned it = 0; it < SPIN; ++it) {
        if (bar_try(b, parity)) return true;
        if ((it & 1023u) == 1023u && *reinterpret_cast<volatile int*>(&bars->fail)) return false;
    }
    *reinterpret_cast<volatile int*>(&bars->fail) = 1;
    return false;
}
__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity, TileBars* bars) {  // the same answer in every lane
    return __all_sync(0xffffffffu, bar_wait(b, parity, bars));
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(su32(bar)) : "memory");
}
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// D (+)= A B, A in tensor memory, B in shared memory (descriptor in two words: what varies, what does not)
template <bool ADD> __device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t b_hi, uint32_t idesc) {
    asm volatile("{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %5, 0;\n mov.b64 db, {%2, %3};\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}\n"
                 ::"r"(d), "r"(a), "r"(b), "r"(b_hi), "r"(idesc), "n"(int(ADD)) : "memory");
}
// a value that every lane of a warp has: the compiler then knows, and keeps loops and MMA operands in uniform registers
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(bar)) : "memory");
}
#define KT_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define KT_I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
__device__ __forceinline__ void tm_ld32(uint32_t a, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
        "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : KT_R8(r, 0), KT_R8(r, 8), KT_R8(r, 16), KT_R8(r, 24) : "r"(a) : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t a, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : KT_R8(r, 0), KT_R8(r, 8) : "r"(a) : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t a, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::KT_I8(r, 0), KT_I8(r, 8), "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t tm_ld1(uint32_t a) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(a) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r)::"memory");
    return r;
}
// Loads return at once; what they bring is there behind the wait. It takes the registers as operands, so that nothing that reads
// them can be moved in front of it.
#define KT_W8(r, o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]), "+r"(r[o + 7])
__device__ __forceinline__ void tm_wait(uint32_t (&r)[16]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : KT_W8(r, 0), KT_W8(r, 8)::"memory"); }
__device__ __forceinline__ void tm_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : KT_W8(r, 0), KT_W8(r, 8), KT_W8(r, 16), KT_W8(r, 24)::"memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_st32(uint32_t a, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
        "%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        ::KT_I8(r, 0), KT_I8(r, 8), KT_I8(r, 16), KT_I8(r, 24), "r"(a) : "memory");
}
// Shared-memory operands with 128-byte swizzle. Keys: 64 rows (N) of 64 values (K) in a row, 8-row groups 1024 bytes apart.
// Values: rows are K (keys), 8-row groups 1024 bytes apart, 64 of the N = 128 dimensions in a row, the others HALF bytes behind.
// Low word: address / 16 and (values) HALF / 16 << 16; high word: 1024 / 16, version 1, swizzle 128.
constexpr uint32_t KT_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t a, uint32_t far) { return ((a & 0x3FFFF) >> 4) | (far >> 4) << 16; }
// fp16 x fp16 -> fp32, M = 128 from tensor memory, N columns; B with N along the rows when `cols`
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool cols) {
    return (1u << 4) | (cols ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(KT_ROWS >> 4) << 24);
}

// two fp32 numbers in one instruction
using Two = unsigned long long;
__device__ __forceinline__ Two two(uint32_t a, uint32_t b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ Two two(float a, float b) { return two(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ float2 parts(Two x) {
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(x));
    return make_float2(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A row's scores of one key tile in tensor memory (128 columns from sp) -> weights in their place, per 16 keys 8 columns of hi and 8
// of lo; running maximum m and denominator l. Returns what earlier sums are to be multiplied by. EDGE: only the first
// `left` keys are seen. The loops stay rolled: straight-line code that a warp runs once per tile comes in at the
// speed of instruction fetch (unrolled, with both forms in one body, this took 3000 clocks a tile).
template <bool EDGE> __device__ __forceinline__ float tile_weights(uint32_t sp, float f, int left, float& m, float& l) {
    float mx = -INFINITY;
#pragma unroll 1
    for (int h = 0; h < KT_KEYS; h += 32) {
        uint32_t x[32];
        tm_ld32(sp + h, x);
        tm_wait(x);
        float u[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            const float x0 = EDGE && i >= left - h ? -INFINITY : __uint_as_float(x[i]);
            const float x1 = EDGE && i + 1 >= left - h ? -INFINITY : __uint_as_float(x[i + 1]);
            u[(i >> 1) & 3] = max3(u[(i >> 1) & 3], x0, x1);
        }
        mx = fmaxf(max3(u[0], u[1], u[2]), u[3]);
    }
    mx = fmaxf(m, mx);
    const float corr = mx == -INFINITY ? 1.f : ex2((m - mx) * f), base = mx == -INFINITY ? 0.f : mx;
    m = mx;
    const Two ff = two(f, f), nb = two(-base, -base), up = two(KA_P, KA_P), minus = two(-1.f, -1.f);
    Two sum = two(0.f, 0.f), sum_b = sum;
    auto weigh = [&](const uint32_t (&x)[16], int h) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const uint32_t x0 = EDGE && i >= left - h ? 0xff800000u : x[i], x1 = EDGE && i + 1 >= left - h ? 0xff800000u : x[i + 1];
            const float2 y = parts(fma2(add2(two(x0, x1), nb), ff, up));
            const float p0 = ex2(y.x), p1 = ex2(y.y);
            const Two pp = two(p0, p1);
            if (i & 2) sum_b = add2(sum_b, pp);
            else sum = add2(sum, pp);
            // hi: the upper 11 bits (exact in fp16 from 2^-14 on, 2^-25 off at most below: weights go up to 2^14); lo: the rest
            const float h0 = __uint_as_float(__float_as_uint(p0) & 0xffffe000u), h1 = __uint_as_float(__float_as_uint(p1) & 0xffffe000u);
            const float2 r = parts(fma2(two(h0, h1), minus, pp));
            const __half2 hi = __floats2half2_rn(h0, h1), lo = __floats2half2_rn(r.x, r.y);
            p[i / 2] = *reinterpret_cast<const uint32_t*>(&hi);
            p[8 + i / 2] = *reinterpret_cast<const uint32_t*>(&lo);
        }
        tm_st16(sp + h, p);
    };
    // The next 16 scores are on their way while 16 are worked on. No load is under way where the loop turns: what a loop
    // carries may be copied there, before the load has come in.
#pragma unroll 1
    for (int h = 0; h < KT_KEYS; h += 64) {
        uint32_t xa[16], xb[16], xc[16], xd[16];
        tm_ld16(sp + h, xa);
        tm_wait(xa);
        tm_ld16(sp + h + 16, xb);
        weigh(xa, h);
        tm_wait(xb);
        tm_ld16(sp + h + 32, xc);
        weigh(xb, h + 16);
        tm_wait(xc);
        tm_ld16(sp + h + 48, xd);
        weigh(xc, h + 32);
        tm_wait(xd);
        weigh(xd, h + 48);
    }
    const float2 t = parts(add2(sum, sum_b));
    l = l * corr + (t.x + t.y);
    tm_wait_st();
    return corr;
}

// consecutive rows of a tile: row, its token and its head among the group's (one division for all of them)
struct RowWalk {
    int row, token, head;
    __device__ __forceinline__ RowWalk(int r, int group) : row(r), token(r / group), head(r % group) {}
    __device__ __forceinline__ void step(int group) {
        ++row;
        if (++head == group) { head = 0; ++token; }
    }
};

// What a CTA works on
struct TileJob {
    int s, j, i, c, kb, ke, vis, vis_min, tiles, edge0;
    KvSeq sq;
    bool cut;
};

template <int PL>
__global__ void __launch_bounds__(KT_THREADS, 1) k_kv_attn_tile(const __grid_constant__ CUtensorMap map, const KvAttnArgs a, int row0,
                                                                int rows_total, int* err) {
    using S = TileShape<PL>;
    extern __shared__ uint8_t tile_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tile_raw) + 1023) & ~uintptr_t(1023));
    TileBars* bars = reinterpret_cast<TileBars*>(smem + S::RING);
    float* ex = reinterpret_cast<float*>(smem + S::RING + 1024);  // [2][128] x 2 words between the teams
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
    TileJob b;
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&bars->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // block -> (tile, key head, split): the last tiles, which see most of a sequence, first; splits fastest
    int64_t bx = blockIdx.x;
    b.c = int(bx % a.splits);
    bx /= a.splits;
    b.j = int(bx % a.HKV);
    const int u = a.tiles_max - 1 - int(bx / a.HKV);
    bool work = kv_tile_of(a, u, &b.s, &b.i);
    int nrows = 0;
    if (work) {
        b.sq = kv_seq(a.rows, b.s);
        nrows = uniform(b.sq.nq * a.group);
        b.vis = uniform(kv_visible(a.rows, b.sq, min(((b.i + 1) * KT_ROWS - 1) / a.group, b.sq.nq - 1)));
        b.vis_min = uniform(kv_visible(a.rows, b.sq, b.i * KT_ROWS / a.group));
        b.cut = a.splits > 1;
        b.kb = b.c * a.chunk;
        b.ke = b.c < a.splits - 1 ? min(b.vis, b.kb + a.chunk) : b.vis;
        work = !b.c || b.kb < b.ke;  // (an empty range: the join does not look at it)
        b.tiles = uniform(max(0, (b.ke - b.kb + KT_KEYS - 1) / KT_KEYS));
        // edge tiles: those with keys that not every row sees, and a last one that ends inside (at most 3)
        b.edge0 = uniform(max(0, min(b.vis_min, b.vis / KT_KEYS * KT_KEYS) - b.kb) / KT_KEYS);
    }
    if (tid == 0) bars->fail = 0;
    bool ok = true;
    auto all_here = [] { asm volatile("bar.sync 0, %0;" ::"n"(KT_THREADS) : "memory"); };
    // Ring elements in the order of use: K0, K1, V0, K2, V1, K3, V2, ...: K of tile n is element 2n - 1 (K0: 0), V is 2n + 2
    // (the last tile's one earlier: no K comes before it)
    auto k_elem = [](int n) { return n == 0 ? 0 : 2 * n - 1; };
    auto v_elem = [&](int n) { return n == b.tiles - 1 ? 2 * n + 1 : 2 * n + 2; };

    if (warp >= 8) {
        // 384 threads start with 168 registers; 128 of them give what the 256 of the rows take: 128 * 80 + 256 * 208 <= 384 * 168
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (work) {
        const int N = b.tiles, edge0 = b.edge0;
        before_sync();
        all_here();
        after_sync();
        if (warp == 8) {  // ---- keys and values
            int issued = 0;
            for (int e = 0; e < 2 * N && ok; ++e) {
                const bool is_v = e == 2 * N - 1 || (e >= 2 && e % 2 == 0);
                const int n = is_v ? (e == 2 * N - 1 ? N - 1 : e / 2 - 1) : (e + 1) / 2;
                const int slot = e % S::SLOTS;
                const uint32_t parity = ((e / S::SLOTS) & 1) ^ 1;
                if (e < S::SLOTS && (slot + 1) * S::SLOT > S::Q_STAGE) {  // the queries pass through here first
                    ok = warp_wait(&bars->q_full, 0, bars);
                    if (!ok) break;
                }
                ok = warp_wait(bars->empty + slot, parity, bars);
                if (!ok) break;
                const int key0 = b.kb + n * KT_KEYS;
                const int box = min(a.rows.page, 64), boxes = (min(KT_KEYS, b.vis - key0) + box - 1) / box;  // pages with visible keys
                if (lane == 0) bar_expect(bars->full + slot, uint32_t(boxes * box * 128 * 2 * PL));
                __syncwarp();
                if (lane < boxes * 2 * PL) {  // a lane per (page, half, plane)
                    const int pl = lane % PL, half = lane / PL % 2, q = lane / PL / 2, key = key0 + q * box;
                    const int pg = kv_page(a.rows, b.s, key);
                    // a page outside the pool: rows behind the pool, which arrive as zeros
                    const int y = pg < 0 ? rows_total
                                         : row0 + int((((int64_t(pg) * 2 + is_v) * a.HKV + b.j) * PL + pl) * a.rows.page) + (key & (a.rows.page - 1));
                    tma_rows(su32(smem + slot * S::SLOT + pl * S::PLANE + half * S::HALF + q * box * 128), &map, half * 64, y, bars->full + slot);
                }
                ++issued;
                if (is_v && n >= edge0) {
                    __syncwarp();
                    if (lane == 0) bar_arrive(bars->go + (n - edge0));
                }
            }
            if (!ok)  // nothing may still be arriving when the CTA ends
                for (int e = max(0, issued - S::SLOTS); e < issued; ++e)
                    for (unsigned it = 0; it < KT_SPIN && !bar_try(bars->full + e % S::SLOTS, (e / S::SLOTS) & 1); ++it) {}
        } else if (warp == 11) {  // ---- values of the edge tiles
            for (int n = edge0; n < N && ok; ++n) {
                const int e = v_elem(n), have = min(KT_KEYS, b.vis - (b.kb + n * KT_KEYS)), up = (have + 15) / 16 * 16;
                // (a parity tells a phase from the one before it only: the slot's turn has come once its load is issued)
                ok = warp_wait(bars->go + (n - edge0), 0, bars) && warp_wait(bars->full + e % S::SLOTS, (e / S::SLOTS) & 1, bars);
                if (!ok) break;
                uint8_t* v = smem + (e % S::SLOTS) * S::SLOT;
                for (int part = 0; part < 2 * PL; ++part)  // rows behind the last key
                    for (int w = lane; w < (up - have) * 8; w += 32) *reinterpret_cast<uint4*>(v + part * S::HALF + have * 128 + w * 16) = make_uint4(0, 0, 0, 0);
                uint32_t any = 0;
                if (b.vis_min < b.vis)
                    for (int part = 0; part < 2 * PL; ++part)
#pragma unroll 8
                        for (int w = lane; w < KT_KEYS * 8; w += 32) {  // an exponent of all ones carries into the sign's place
                            const uint4 u = *reinterpret_cast<const uint4*>(v + part * S::HALF + w * 16);
                            const uint32_t c = (((u.x & 0x7c007c00u) + 0x04000400u) | ((u.y & 0x7c007c00u) + 0x04000400u) |
                                                ((u.z & 0x7c007c00u) + 0x04000400u) | ((u.w & 0x7c007c00u) + 0x04000400u)) & 0x80008000u;
                            any |= w < have * 8 ? c : 0u;
                        }
                const bool odd = __any_sync(0xffffffffu, any != 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    bars->odd[n - edge0] = odd;
                    bar_arrive(bars->edge + (n - edge0));
                }
            }
        } else {  // ---- MMA issuers, one per team: the whole warp walks the team's tiles, one lane issues
            // (with all of it inside `if (lane == 0)` every operand went through a vector register: 100 clocks per MMA). An MMA is
            // issued about when it starts, so a wait between two of them is time that the tensor core stands still: with an
            // issuer per team one waits while the other's products run. O(n) and S(n + 2) follow one another without a wait.
            constexpr uint32_t id_s = idesc_f16(KT_KEYS, false), id_o = idesc_f16(KV_D, true);
            const int w = warp - 9;
            const uint32_t ring_k = desc_lo(su32(smem), 0), ring_v = desc_lo(su32(smem), S::HALF);
            const uint32_t s_at = 128 + w * 128, o_at = 384;
            auto scores = [&](int n) {
                const int slot = k_elem(n) % S::SLOTS;
                const uint32_t k = ring_k + slot * (S::SLOT >> 4);
                if (elect()) {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const uint32_t at = k + (ks >> 2) * (S::HALF >> 4) + (ks & 3) * 2;
                        if (ks == 0) mma_ts<false>(s_at, 64, at, KT_DESC_HI, id_s);
                        else mma_ts<true>(s_at, 64 + ks * 8, at, KT_DESC_HI, id_s);
                        if (PL == 2) mma_ts<true>(s_at, ks * 8, at + (S::PLANE >> 4), KT_DESC_HI, id_s);
                    }
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) mma_ts<true>(s_at, ks * 8, k + (ks >> 2) * (S::HALF >> 4) + (ks & 3) * 2, KT_DESC_HI, id_s);
                    commit(bars->empty + slot);
                    commit(bars->s_full + w);
                }
                __syncwarp();
            };
            auto k_wait = [&](int n) {
                const int e = k_elem(n);
                return warp_wait(bars->full + e % S::SLOTS, (e / S::SLOTS) & 1, bars);
            };
            if (w < N) {
                ok = warp_wait(&bars->q_full, 0, bars) && k_wait(w);
                after_sync();
                if (ok) scores(w);
            }
            for (int n = w; n < N && ok; n += 2) {
                const bool more = n + 2 < N;
                const int e = v_elem(n), slot = e % S::SLOTS;
                // Weights, values and (F16) the keys behind them in one wait, a lane each: a wait costs 200 clocks even when all
                // is there. A wait for a slot is good only when the load before it in that slot is known to have come in (a parity
                // tells two neighbouring phases apart, no more); the weights being ready says so, hence the second look at all.
                {
                    const int ek = k_elem(n + 2);
                    uint64_t* bar = bars->pv_ready + w;
                    uint32_t par = uint32_t(n >> 1) & 1;
                    if (lane & 1) { bar = bars->full + slot; par = (e / S::SLOTS) & 1; }
                    if (PL == 1 && more && (lane & 2)) { bar = bars->full + ek % S::SLOTS; par = (ek / S::SLOTS) & 1; }
                    if (n >= edge0 && lane >= 16) { bar = bars->edge + (n - edge0); par = 0; }
                    ok = warp_wait(bar, par, bars) && warp_wait(bar, par, bars);
                }
                if (!ok) break;
                after_sync();
                const uint32_t v = ring_v + slot * (S::SLOT >> 4);
                const int steps = min(KT_KEYS / 16, (b.vis - (b.kb + n * KT_KEYS) + 15) / 16);
                if (elect()) {
#pragma unroll
                    for (int ks = 0; ks < KT_KEYS / 16; ++ks) {  // weights of 16 keys: 8 columns of hi, 8 of lo
                        if (ks >= steps) break;
                        if (ks == 0) mma_ts<false>(o_at, s_at + 8, v, KT_DESC_HI, id_o);
                        else mma_ts<true>(o_at, s_at + ks * 16 + 8, v + ks * 128, KT_DESC_HI, id_o);
                        if (PL == 2) mma_ts<true>(o_at, s_at + ks * 16, v + (S::PLANE >> 4) + ks * 128, KT_DESC_HI, id_o);
                    }
#pragma unroll
                    for (int ks = 0; ks < KT_KEYS / 16; ++ks) {
                        if (ks >= steps) break;
                        mma_ts<true>(o_at, s_at + ks * 16, v + ks * 128, KT_DESC_HI, id_o);
                    }
                    commit(bars->empty + slot);
                    commit(bars->o_full + w);
                }
                __syncwarp();
                if (more) {
                    if (PL == 2) {  // (three slots: its load has waited for the product before this one)
                        ok = k_wait(n + 2);
                        after_sync();
                    }
                    if (ok) scores(n + 2);
                }
            }
        }
        __syncwarp();
        before_sync();
        all_here();
        after_sync();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        if (work) {
        const int N = b.tiles, edge0 = b.edge0;
            // queries: a warp copies 16 whole rows into the end of the ring, then every thread takes half of its row to tensor
            // memory as hi | lo (a thread per row straight from global memory: 10000 clocks)
            const RowWalk first(b.i * KT_ROWS + warp * 16, a.group);
            float* qs = reinterpret_cast<float*>(smem + S::Q_STAGE);  // [row][KT_LD]
            {
                RowWalk w = first;
#pragma unroll 4
                for (int q = 0; q < 16; ++q, w.step(a.group)) {
                    const bool on = w.row < nrows;
                    cp16z(su32(qs + (warp * 16 + q) * KT_LD + lane * 4),
                          on ? a.q + (b.sq.row0 + w.token) * a.ldq + (b.j * a.group + w.head) * KV_D + lane * 4 : a.q, on);
                }
            }
        if (tid == 0) {
            for (int s = 0; s < S::SLOTS; ++s) { bar_init(bars->full + s, 1); bar_init(bars->empty + s, 1); }
            for (int w = 0; w < 2; ++w) { bar_init(bars->s_full + w, 1); bar_init(bars->pv_ready + w, 8); bar_init(bars->o_full + w, 1); }
            bar_init(&bars->q_full, 8);
            for (int k = 0; k < KT_MAXEDGE; ++k) { bar_init(bars->go + k, 1); bar_init(bars->edge + k, 1); }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        before_sync();
        all_here();
        after_sync();
        {  // ---- two teams: rows
            const int team = warp >> 2, r = (warp & 3) * 32 + lane, row = b.i * KT_ROWS + r;
            const uint32_t mine = uint32_t((warp & 3) * 32) << 16;  // (all 512 columns are this CTA's: they start at 0)
            const bool real = row < nrows;
            const int see = real ? kv_visible(a.rows, b.sq, row / a.group) : b.vis;
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("bar.sync 1, 256;" ::: "memory");
            float f;
            {
                float4 x[16];
                float mx = 0.f;
#pragma unroll
                for (int u = 0; u < 16; ++u) {
                    x[u] = *reinterpret_cast<const float4*>(qs + r * KT_LD + team * 64 + 4 * u);
                    mx = max3(mx, max3(fabsf(x[u].x), fabsf(x[u].y), fabsf(x[u].z)), fabsf(x[u].w));
                }
                ex[team * 128 + r] = mx;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                const RowScale rs = row_scale(fmaxf(ex[r], ex[128 + r]), a.scale2);
                f = rs.f;
                const Two k1 = two(rs.up.s1, rs.up.s1), k2 = two(rs.up.s2, rs.up.s2);
                uint32_t hi[32], lo[32];
#pragma unroll
                for (int u = 0; u < 16; ++u) {
                    const float2 y = parts(mul2(mul2(two(x[u].x, x[u].y), k1), k2)), z = parts(mul2(mul2(two(x[u].z, x[u].w), k1), k2));
                    half_pair_finite(y.x, y.y, hi[2 * u], lo[2 * u]);  // (an infinity becomes infinity and NaN: its row is NaN either way)
                    half_pair_finite(z.x, z.y, hi[2 * u + 1], lo[2 * u + 1]);
                }
                tm_st32(mine + team * 32, hi);
                tm_st32(mine + 64 + team * 32, lo);
            }
            tm_wait_st();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // TMA may write here now
            before_sync();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars->q_full);
            Two O[KV_D / 2];
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int d = 0; d < KV_D / 2; ++d) O[d] = two(0.f, 0.f);
            const uint32_t sp = mine + 128 + team * 128, so = mine + 384;
            if (team == 1 && lane == 0) bar_arrive(bars->pv_ready);  // O is free at first
#pragma unroll 1
            for (int n = team; n < N; n += 2) {
                ok = warp_wait(bars->s_full + team, (n >> 1) & 1, bars);
                if (!ok) break;
                after_sync();
                bool odd = false;
                float corr;
                if (n < edge0) {
                    corr = tile_weights<false>(sp, f, KT_KEYS, m, l);
                } else {
                    const int left = see - (b.kb + n * KT_KEYS);  // keys of the tile that the row sees
                    corr = tile_weights<true>(sp, f, left, m, l);
                    ok = warp_wait(bars->edge + (n - edge0), 0, bars);
                    if (!ok) break;
                    odd = *reinterpret_cast<volatile int*>(bars->odd + (n - edge0)) != 0;
                    if (odd) {  // key by key, for the rows that see it
                        const int e = v_elem(n);
                        ok = warp_wait(bars->full + e % S::SLOTS, (e / S::SLOTS) & 1, bars);
                        if (!ok) break;
                        const uint8_t* v = smem + (e % S::SLOTS) * S::SLOT;
                        const Two cc = two(corr, corr), zero = two(0.f, 0.f);
#pragma unroll
                        for (int d = 0; d < KV_D / 2; ++d) O[d] = fma2(O[d], cc, zero);
#pragma unroll 1
                        for (int key = 0; key < KT_KEYS; ++key) {
                            __syncwarp();
                            const uint32_t at = sp + (key >> 4) * 16 + ((key & 15) >> 1), sh = (key & 1) * 16;
                            const float w = h2f_bits((tm_ld1(at) >> sh) & 0xffffu) + h2f_bits((tm_ld1(at + 8) >> sh) & 0xffffu);
                            if (key >= left) continue;
                            const Two ww = two(w, w);
#pragma unroll
                            for (int d = 0; d < KV_D; d += 2) {
                                const int off = (d >> 6) * S::HALF + key * 128 + ((((d & 63) >> 3) ^ (key & 7)) << 4) + (d & 7) * 2;
                                float2 u = __half22float2(*reinterpret_cast<const __half2*>(v + off));
                                if (PL == 2) {
                                    const float2 u2 = __half22float2(*reinterpret_cast<const __half2*>(v + S::PLANE + off));
                                    u.x += u2.x; u.y += u2.y;
                                }
                                O[d / 2] = fma2(ww, two(u.x, u.y), O[d / 2]);
                            }
                        }
                        __syncwarp();
                    }
                }
                before_sync();
                __syncwarp();
                if (lane == 0) bar_arrive(bars->pv_ready + team);
                ok = warp_wait(bars->o_full + team, (n >> 1) & 1, bars);  // (a barrier per team: a wait that skips phases would take an old one for its own)
                if (!ok) break;
                after_sync();
                if (!odd) {  // the next 32 sums are on their way while these are added
                    const Two cc = two(corr, corr);
                    uint32_t x[2][32];
                    tm_ld32(so, x[0]);
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        tm_wait(x[h & 1]);
                        if (h < 3) tm_ld32(so + h * 32 + 32, x[(h + 1) & 1]);
#pragma unroll
                        for (int i = 0; i < 32; i += 2) O[h * 16 + i / 2] = fma2(O[h * 16 + i / 2], cc, two(x[h & 1][i], x[h & 1][i + 1]));
                    }
                }
                before_sync();
                __syncwarp();
                if (lane == 0) bar_arrive(bars->pv_ready + (team ^ 1));  // O is free for the other team's next product
            }
            // the teams' results: through shared memory (the ring is used up once both are here)
            ex[256 + (team * 128 + r) * 2] = m;
            ex[257 + (team * 128 + r) * 2] = l;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const float m0 = ex[256 + r * 2], l0 = ex[257 + r * 2], m1 = ex[512 + r * 2], l1 = ex[513 + r * 2];
            const float M = fmaxf(m0, m1), k0 = M == -INFINITY ? 1.f : ex2((m0 - M) * f), k1 = M == -INFINITY ? 1.f : ex2((m1 - M) * f);
            const float den = k0 * l0 + k1 * l1, k = team ? k1 : k0;
            const bool final_here = !b.cut || b.vis <= a.chunk;
            const float inv = final_here ? (den == 0.f ? 0.f : 1.f / den) : 1.f;
            float* stage = reinterpret_cast<float*>(smem);  // [team][row][KT_LD]
            float4* own_row = reinterpret_cast<float4*>(stage + (team * KT_ROWS + r) * KT_LD);
            const float ki = k * inv;
#pragma unroll
            for (int d = 0; d < KV_D; d += 4) {
                const float2 x = parts(O[d / 2]), y = parts(O[d / 2 + 1]);
                own_row[d / 4] = make_float4(x.x * ki, x.y * ki, y.x * ki, y.y * ki);
            }
            const int64_t slot = (int64_t(u) * a.HKV + b.j) * a.splits + b.c;
            float* part = a.part + slot * KT_ROWS * KA_ROW;
            if (!final_here && team == 0) { part[KT_ROWS * KV_D + r] = M; part[KT_ROWS * (KV_D + 1) + r] = den; part[KT_ROWS * (KV_D + 2) + r] = f; }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (ok) {
                RowWalk w = first;
                bool odd = false;  // some result may be NaN
#pragma unroll 4
                for (int q = warp * 16; q < warp * 16 + 16; ++q, w.step(a.group)) {
                    const float4 x = *reinterpret_cast<const float4*>(stage + q * KT_LD + lane * 4);
                    const float4 y = *reinterpret_cast<const float4*>(stage + (KT_ROWS + q) * KT_LD + lane * 4);
                    float* dst = final_here ? a.out + (b.sq.row0 + w.token) * a.ldo + (b.j * a.group + w.head) * KV_D : part + q * KV_D;
                    const float4 z = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
                    if (w.row < nrows) *reinterpret_cast<float4*>(dst + lane * 4) = z;
                    odd |= !((z.x + z.y) + (z.z + z.w) < INFINITY);
                }
                if (final_here && __any_sync(0xffffffffu, odd)) {
                    w = first;
#pragma unroll 1
                    for (int q = warp * 16; q < warp * 16 + 16 && w.row < nrows; ++q, w.step(a.group)) {
                        const float most = fmaxf(ex[256 + q * 2], ex[512 + q * 2]), sums = ex[257 + q * 2] + ex[513 + q * 2];
                        if (!(sums > 0.f) || most == -INFINITY) continue;  // (its scores are not finite)
#pragma unroll 1
                        for (int d = lane * 4; d < lane * 4 + 4; ++d) {
                            const float z = stage[q * KT_LD + d] + stage[(KT_ROWS + q) * KT_LD + d];
                            if (z != z)
                                a.out[(b.sq.row0 + w.token) * a.ldo + (b.j * a.group + w.head) * KV_D + d] =
                                    kv_not_finite(a, b.s, b.j, kv_visible(a.rows, b.sq, w.token), d);
                        }
                    }
                }
            }
        }
        before_sync();
        all_here();
        after_sync();
        }
    }
    all_here();
    if (tid == 0 && bars->fail) atomicExch(err, 1);
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(bars->tmem) : "memory");
}

// The bounded wait on a barrier that nobody arrives at, with a short limit: it must give up and raise the error word
__global__ void k_kv_wait_expiry(int* err) {
    __shared__ TileBars bars;
    if (threadIdx.x == 0) {
        bars.fail = 0;
        bar_init(&bars.q_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (!bar_wait<1u << 12>(&bars.q_full, 0, &bars) && bars.fail) atomicExch(err, 1);
    }
}

struct TilePlan { int64_t tiles; int splits, chunk; };

// few_max: sequences of up to so many query rows belong to the narrow kernel
TilePlan tile_plan(const Kv* kv, const elb_kv_batch* b, int n_head, int few_max) {
    TilePlan p{};
    const int64_t rows = int64_t(b->n_tok) * (n_head / kv->HKV);
    // tiles of 128 rows: whatever the sequences' lengths are, each adds at most one that is not full
    p.tiles = b->n_seq == 1 ? (rows + KT_ROWS - 1) / KT_ROWS : rows / KT_ROWS + std::min<int64_t>(b->n_seq, rows / (few_max + 1));
    // The cut of the keys. A CTA's start and end cost as much as 5 to 8 tiles of keys, so its range should be long, at least 4 tiles;
    // but a second wave of CTAs costs as much as the first. When the sequences have about as many rows each, their tiles are
    // known and the ranges are made for one wave; when not (lengths will differ as well, and short ones leave early), half of the
    // sequences' last tiles are counted and the ranges are made for one and a half. Cut in 1, 2, 3, 4, 6 ranges, us, F16: 9 sequences
    // of 64 tokens at 4096 keys, 16 heads on 8 (72 CTAs) 76, 56, 76, 70, 83; 2 of 64 at 8000, 32 on 8 (32) 154, 93, 69, 59, 80; 3 of
    // 300 at 2000 (240) 93, 126, 133, 148, 169; 9 of 3-77 at 203-4100, 16 on 8 65, 53, 49, 52, 59; 4 of 20-300 at 300-3000 66, 85,
    // 91, 85, 105. (All key tiles dealt out evenly over one CTA per SM, which walks from tile to tile, with a launch before
    // and a join behind: 73, -, 123, -, -.)
    const int64_t most_q = std::max(1, std::min(b->max_q, b->n_tok));
    const bool alike = 4 * int64_t(b->n_tok) >= 3 * b->n_seq * most_q;
    const int64_t likely = std::min(b->n_seq * ((most_q * (n_head / kv->HKV) + KT_ROWS - 1) / KT_ROWS), rows / KT_ROWS + (b->n_seq + 1) / 2);
    const int64_t base = kv->HKV * std::max<int64_t>(1, b->n_seq == 1 ? p.tiles : std::min(p.tiles, likely));
    const int len = kv_most(kv, b);
    int64_t want = std::max<int64_t>(1, alike ? kv->sm_count / base : (3 * kv->sm_count + base) / (2 * base));
    want = std::min<int64_t>(want, (len + 4 * KT_KEYS - 1) / (4 * KT_KEYS));
    p.chunk = int((len + want - 1) / want + KT_KEYS - 1) / KT_KEYS * KT_KEYS;
    p.splits = (len + p.chunk - 1) / p.chunk;
    return p;
}

}  // namespace

int kv_attn_tile_prepare() {
    ELB_TRY(ensure_dyn_smem(reinterpret_cast<const void*>(k_kv_attn_tile<1>), TileShape<1>::SMEM));
    return ensure_dyn_smem(reinterpret_cast<const void*>(k_kv_attn_tile<2>), TileShape<2>::SMEM);
}

int kv_attention_check(const Kv* kv) {
    if (*reinterpret_cast<volatile int*>(kv->err)) {
        *kv->err = 0;
        return fail(ELB_ERR_CUDA, "kv_attention: a bounded wait ran out in an earlier call");
    }
    return ELB_OK;
}

int kv_attention_wait_expiry(const Kv* kv) {  // kv_attention_check() behind a synchronize reports it
    k_kv_wait_expiry<<<1, 32>>>(kv->err_dev);
    ELB_CUDA(cudaGetLastError());
    ELB_CUDA(cudaStreamSynchronize(nullptr));
    return ELB_OK;
}

size_t kv_attn_tile_work(const Kv* kv, const elb_kv_batch* b, int n_head, int few_max) {
    const TilePlan p = tile_plan(kv, b, n_head, few_max);
    if (p.splits == 1) return 0;
    return size_t(p.tiles) * kv->HKV * p.splits * KT_ROWS * KA_ROW * 4;
}

int kv_attn_tile_launch(const Kv* kv, int layer, KvAttnArgs a, const elb_kv_batch* b, cudaStream_t s) {
    const TilePlan p = tile_plan(kv, b, a.H, a.few_max);
    const int64_t blocks = p.tiles * kv->HKV;
    if (blocks * p.splits > 0x7fffffff || blocks * KT_ROWS / 8 > 0x7fffffff) return fail(ELB_ERR_UNSUPPORTED, "kv_attention: too many rows");
    if (blocks == 0) return ELB_OK;
    a.splits = p.splits; a.chunk = p.chunk; a.tiles_max = int(p.tiles);
    const int64_t layer_rows = kv->layer_halves() / KV_D;
    auto run = [&](auto kernel, int smem) -> int {
        kernel<<<unsigned(blocks * p.splits), KT_THREADS, smem, s>>>(kv->map, a, int(layer * layer_rows), int(kv->n_layer * layer_rows), kv->err_dev);
        ELB_CUDA(cudaGetLastError());
        return ELB_OK;
    };
    if (kv->planes == 1) ELB_TRY(run(k_kv_attn_tile<1>, TileShape<1>::SMEM));
    else ELB_TRY(run(k_kv_attn_tile<2>, TileShape<2>::SMEM));
    return p.splits > 1 ? kv_attn_join(a, KT_ROWS, blocks, s) : ELB_OK;
}

}  // namespace elb
