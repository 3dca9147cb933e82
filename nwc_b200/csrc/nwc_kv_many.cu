/* Attention of many query rows (a prompt chunk, a large draft tree) over a cache of nwc_kv.h on the 5th-generation tensor
 * cores.  What a token sees: see nwc_kv_attention.cu.
 *
 * All query heads of a key/value head are rows of one matrix (row = token * group + head), so K and V are read once for the
 * group.  A CTA holds two tiles of 128 rows ("streams") and walks over tiles of 128 keys: S = Q K^T into tensor memory, 128
 * threads per stream turn their row of S into weights P (one thread = one row: no shuffles), P goes back to tensor memory as
 * the A operand of O += P V.  While one stream's weights are computed the tensor cores work for the other:
 *
 *   tensor:   S0(j+1)  PV1(j) S1(j+1)   PV0(j+1) S0(j+2) ...
 *   stream 0:      weights of S0(j+1)
 *   stream 1:                  weights of S1(j+1)
 *
 * With at most 128 rows in all, both streams hold the same rows and take the key tiles in turn; their shares meet at the end.
 * Few rows over a long cache: the keys are divided over several CTAs and joined by a second kernel.
 *
 * Bound: 4 * 128 * 128 * head_dim multiply-adds per pair of tiles on the tensor cores (2048 clocks at head_dim 128), and as
 * many clocks of the exponential unit (16 per SM and clock) for 2 * 128 * 128 weights.
 *
 * Roles: warps 0-3 and 4-7 weights of stream 0 and 1 (they also load Q, rescale and write out O), the next four or eight
 * bring K and V into shared memory, one thread behind them issues the MMAs.  A tile
 * of the list of keys may begin, end and wrap anywhere in the ring; a row that is no key of the call is written as zeros
 * (whatever its slot holds, weight 0 times it must be 0).  Whole bf16 tiles are tensor-map copies; e4m3 rows become bf16 on
 * the way, exactly: code and unit have fewer bits than a bf16 number.  All waits are
 * bounded; a role that gives up says so in both status words and stops, the others run out, copies and products in flight are
 * awaited, tensor memory is freed.
 *
 * O is rescaled in tensor memory only when a row's maximum passes the one it is scaled by by more than 2^8 (weights stay below
 * 2^8, sums are fp32): after the first tiles hardly ever.  P is rounded to bf16 (2^-8 relative), the sum of the weights is not.
 */
#include <atomic>
#include <cuda.h>
#include "nwc_kv.h"
#include "nwc_async.cuh"
#include "nwc_launch.h"

namespace nwc {

namespace {

constexpr uint32_t kManyRows = 128u, kManyKeys = 128u;

template <int HD, int ELEM> struct Many {
    static constexpr uint32_t kTile = kManyKeys * HD * 2u, kHalfBytes = kManyKeys * 128u;      /* a bf16 tile: halves of 64 dimensions, 128-byte rows, swizzled */
    /* Operand slots.  Both streams' products with a tile must end before its slot is filled again, and the filling itself takes
       a while, so three slots run dry: the products wait for V, V for the slot, the slot for the products. */
    static constexpr uint32_t kSlots = HD == 64 ? 8u : 5u;
    /* Registers: the 16 warps start with 65536 / 512 = 128 each; those that hold a row of scores take what the others give back:
       8 x 184 + 4 x 72 + 4 x 72 = 16 x 128 (bf16: the producers only start copies), 8 x 168 + 4 x 112 + 4 x 64 = 16 x 128 (e4m3:
       they hold two sets of codes; at 176 / 96 / 64 the tree of 64 over 32768 takes 107 us instead of 90; these forms spill 66 to 78
       bytes). */
    static constexpr uint32_t kProducers = 128u, kMmaWarp = 8u + kProducers / 32u, kThreads = 256u + kProducers + 128u;
    static constexpr int kRegsWeights = ELEM == kKvE4m3 ? 168 : 184, kRegsProduce = ELEM == kKvE4m3 ? 112 : 72, kRegsMma = ELEM == kKvE4m3 ? 64 : 72;
    static constexpr uint32_t kQ = 0u, kRing = 2u * kTile, kBars = kRing + kSlots * kTile;
    static constexpr uint32_t kSmem = 1024u + kBars + (2u * kSlots + 8u) * 8u + 16u;
};

/* shared-memory descriptor, 128-byte swizzle, groups of eight rows 1024 bytes apart: address (in 16 bytes) and leading offset in
   the low word, the rest in the high one */
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lead_bytes) { return ((addr & 0x3FFFFu) >> 4) | ((lead_bytes >> 4) << 16); }
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__host__ __device__ constexpr uint32_t idesc_bf16(uint32_t M, uint32_t N, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major ? 1u << 16 : 0u) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk) { return row * 128u + ((chunk ^ (row & 7u)) << 4); }
__device__ __forceinline__ void sts128u(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) { asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory"); }
/* one arrival for the warp (32 arrivals of single lanes queue up at the barrier: a tile took a thousand clocks longer) */
__device__ __forceinline__ void arrive_warp(uint32_t bar) { __syncwarp(); if ((threadIdx.x & 31u) == 0u) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory"); }
__device__ __forceinline__ void copies_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
/* one box of 64 dimensions x 128 rows of this GPU's own memory into this CTA's shared memory; x is 0 or 64 elements = 128 bytes */
__device__ __forceinline__ void tensor_load(uint32_t dst, const CUtensorMap *map, uint32_t x, uint32_t row, uint32_t plane, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(row), "r"(plane), "r"(bar) : "memory");
}
/* The issuing warp stays together and all of its lanes hold the same descriptors, so that they live in uniform registers; one
   elected lane (`leader`) issues.  (One lane in a branch of its own moves every operand over for each MMA: measured 110
   clocks an MMA that takes 64.) */
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p;
}
__device__ __forceinline__ void mma_commit(uint32_t leader, uint32_t bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(leader) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\tmov.b64 x, {%1, %6};\n\tmov.b64 y, {%2, %6};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(leader), "r"(kDescHigh) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\tmov.b64 y, {%2, %6};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(leader), "r"(kDescHigh) : "memory");
}
__device__ __forceinline__ void tm_load32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
                   "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(addr) : "memory");
}
__device__ __forceinline__ void tm_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_store16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tm_load8(uint32_t addr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tm_store8(uint32_t addr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
/* names registers that a wait has made valid, so that nothing reads them above it (no instruction) */
template <int N> __device__ __forceinline__ void tm_hold(uint32_t (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; e++) asm volatile("" : "+r"(v[e]));
}
/* two fp32 operations in one instruction */
__device__ __forceinline__ uint64_t pack2(float a, float b) { uint64_t d; asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b)); return d; }
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ void tm_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { uint32_t d; asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a)); return d; }
__device__ __forceinline__ void kv_dependency_sync() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
/* One row's scores of a tile -> weights: running maximum m (log2) and sum l updated, P (bf16) over the scores' first columns,
   O rescaled where m was raised.  The 128 scores are in registers throughout. */
template <bool WHOLE>
__device__ __forceinline__ void weights(float scale, uint32_t tm_s, uint32_t tm_o, uint32_t hd, bool have_o, const uint32_t (&vis)[4], float &m, float &l) {
    uint32_t v[4][32];
#pragma unroll
    for (uint32_t ch = 0; ch < 4u; ch++) tm_load32(tm_s + ch * 32u, v[ch]);
    tm_wait_load();
#pragma unroll
    for (uint32_t ch = 0; ch < 4u; ch++) tm_hold(v[ch]);
    float top4[4];
#pragma unroll
    for (uint32_t ch = 0; ch < 4u; ch++) {
        if (!WHOLE) {
#pragma unroll
            for (uint32_t e = 0; e < 32u; e++) if (!((vis[ch] >> e) & 1u)) v[ch][e] = 0xFF800000u;
        }
        float t = __uint_as_float(v[ch][0]);
#pragma unroll
        for (uint32_t e = 1; e < 31u; e += 2u) t = fmaxf(t, fmaxf(__uint_as_float(v[ch][e]), __uint_as_float(v[ch][e + 1])));
        top4[ch] = fmaxf(t, __uint_as_float(v[ch][31]));
    }
    const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * scale;
    const bool raise = top > m + 8.f;
    if (__any_sync(0xffffffffu, raise)) {
        const float up = raise ? top : m, f = up == -INFINITY ? 1.f : exp2_fast(m - up);
        m = up; l *= f;
        if (have_o) {
            for (uint32_t c = 0; c < hd; c += 8u) {                                     /* (rare; few registers beside the scores) */
                uint32_t o[8];
                tm_load8(tm_o + c, o);
                tm_wait_load();
                tm_hold(o);
#pragma unroll
                for (uint32_t e = 0; e < 8u; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tm_store8(tm_o + c, o);
            }
        }
    }
    const float below = m == -INFINITY ? 0.f : -m;
    const uint64_t scale2 = pack2(scale, scale), below2 = pack2(below, below);
    uint64_t sum0 = 0ull, sum1 = 0ull;
#pragma unroll
    for (uint32_t ch = 0; ch < 4u; ch++) {
        uint32_t p[16];
#pragma unroll
        for (uint32_t e = 0; e < 32u; e += 4u) {
            float y0, y1, y2, y3;
            unpack2(fma2(pack2(__uint_as_float(v[ch][e]), __uint_as_float(v[ch][e + 1])), scale2, below2), y0, y1);
            unpack2(fma2(pack2(__uint_as_float(v[ch][e + 2]), __uint_as_float(v[ch][e + 3])), scale2, below2), y2, y3);
            y0 = exp2_fast(y0); y1 = exp2_fast(y1); y2 = exp2_fast(y2); y3 = exp2_fast(y3);
            sum0 = add2(sum0, pack2(y0, y1)); sum1 = add2(sum1, pack2(y2, y3));
            p[e >> 1] = pack_bf16(y0, y1); p[(e >> 1) + 1u] = pack_bf16(y2, y3);
        }
        tm_store16(tm_s + ch * 16u, p);
    }
    float s0, s1;
    unpack2(add2(sum0, sum1), s0, s1);
    l += s0 + s1;
}
/* bits [lo, hi) of a word whose bit 0 is number 0; lo and hi may lie anywhere */
__device__ __forceinline__ uint32_t bit_range(int32_t lo, int32_t hi) {
    lo = max(lo, 0); hi = min(hi, 32);
    if (lo >= hi) return 0u;
    return (0xFFFFFFFFu >> (32 - (hi - lo))) << lo;
}

/* a warp that gave up waiting says so in the call's status word too: its outputs, or its share of them, were not written */
__device__ __forceinline__ void report_wait(bool alive, int *status) { if (!alive && (threadIdx.x & 31u) == 0u) atomicOr(status, kKvStatusWait); }

}  // namespace

template <int HD, int ELEM>
__global__ void __launch_bounds__(Many<HD, ELEM>::kThreads, 1) kv_attention_many_kernel(const KvAttention a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using F = Many<HD, ELEM>;
    constexpr uint32_t NS = F::kSlots, kProducers = F::kProducers;
    extern __shared__ uint8_t many_raw[];
    const uint32_t base = (smem_addr(many_raw) + 1023u) & ~1023u;
    const uint32_t bars = base + F::kBars, full = bars, empty = bars + NS * 8u, q_full = bars + 2u * NS * 8u, s_full = q_full + 16u, p_full = s_full + 16u, o_full = p_full + 16u, tmem_slot = o_full + 16u;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    /* the first `pairs` units are two row tiles, the others one (see the launcher) */
    const uint32_t group = a.n_q / a.c.n_kv, rows = a.T * group, unit = blockIdx.x, split = blockIdx.y;
    const uint32_t kvh = unit % a.c.n_kv, row0 = unit < a.pairs ? unit / a.c.n_kv * 2u * kManyRows : a.pairs / a.c.n_kv * 2u * kManyRows + (unit - a.pairs) / a.c.n_kv * kManyRows;
    const bool solo = unit >= a.pairs || rows - row0 <= kManyRows;
    const uint32_t my_rows = solo ? kManyRows : 2u * kManyRows;
    if (warp == F::kMmaWarp) {
        if (lane == 0) {
            for (uint32_t s = 0; s < NS; s++) { mbar_init(full + s * 8u, kProducers / 32u); mbar_init(empty + s * 8u, 1u); }
            for (uint32_t s = 0; s < 2u; s++) { mbar_init(q_full + s * 8u, 4u); mbar_init(s_full + s * 8u, 1u); mbar_init(p_full + s * 8u, 4u); mbar_init(o_full + s * 8u, 1u); }
            mbar_init_fence();
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    kv_dependency_sync();
    const int32_t pos = *a.pos;
    const bool pos_ok = pos >= 0 && (uint64_t)pos + a.T <= (a.c.window ? 0x7FFFFFFFu : a.c.capacity);
    tm_fence_before();
    __syncthreads();
    tm_fence_after();
    uint32_t tmem; asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
    /* the keys that this CTA's tokens see: as kv_span, for their positions; list index = lead sinks, then positions from first */
    const uint32_t t_first = row0 / group, t_last = min(a.T - 1u, (row0 + my_rows - 1u) / group);
    KvSpan span{0u, 0u, 0u};
    if (pos_ok) span = a.visible ? kv_span(pos, a.T, a.c.window, a.c.sinks) : kv_span((uint32_t)pos + t_first, t_last - t_first + 1u, a.c.window, a.c.sinks);
    const uint32_t slot_first = kv_slot(span.first, a.c.capacity, a.c.window, a.c.sinks), ring = a.c.capacity - a.c.sinks;
    const uint32_t all = (span.count + kManyKeys - 1u) / kManyKeys, tile0 = (uint32_t)((uint64_t)all * split / a.splits), n = (uint32_t)((uint64_t)all * (split + 1u) / a.splits) - tile0;
    /* items of the operand ring: K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1) */
    auto item_k = [](uint32_t t) { return t ? 2u * t - 1u : 0u; };
    auto item_v = [n](uint32_t t) { return t + 1u < n ? 2u * t + 2u : 2u * n - 1u; };
    bool alive = true;
    if (warp < 8u) {
        /* ---- weights ---- */
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F::kRegsWeights));
        const uint32_t s = warp >> 2, wt = tid & 127u, q_tile = solo ? 0u : s, my_row0 = row0 + q_tile * kManyRows;
        const uint32_t my_n = solo ? (s ? n / 2u : (n + 1u) / 2u) : n;                 /* tiles of this stream */
        if (n && !(solo && s)) {
            /* Q: 16 bytes per thread (all loads in flight together), rows beyond the last as zeros */
            constexpr uint32_t kQChunks = HD / 8u, kQPasses = kManyRows * kQChunks / 128u, kQRows = 128u / kQChunks;
            const uint32_t qr = wt / kQChunks, qc = wt % kQChunks;
            uint4 w[kQPasses];
#pragma unroll
            for (uint32_t e = 0; e < kQPasses; e++) {
                const uint32_t row = my_row0 + qr + e * kQRows;
                w[e] = make_uint4(0u, 0u, 0u, 0u);
                if (row < rows) w[e] = *reinterpret_cast<const uint4 *>(a.q + (uint64_t)(row / group) * a.ldq + (uint64_t)(kvh * group + row % group) * HD + qc * 8u);
            }
#pragma unroll
            for (uint32_t e = 0; e < kQPasses; e++) sts128u(base + F::kQ + q_tile * F::kTile + (qc >> 3) * F::kHalfBytes + swizzled(qr + e * kQRows, qc & 7u), w[e].x, w[e].y, w[e].z, w[e].w);
            async_proxy_fence();
            arrive_warp(q_full + q_tile * 8u);
        }
        const uint32_t row = my_row0 + wt, row_ok = row < rows, token = min(row, rows - 1u) / group, idx_pos = (uint32_t)pos - span.first + span.lead;      /* (tree) list index of the first draft */
        const uint32_t own = (uint32_t)pos + (a.depth ? (uint32_t)a.depth[token] : token), words = (a.T + 31u) / 32u;
        /* in list indices this row sees [lo, hi) and what lies below `always` of it */
        const int32_t hi = a.visible ? (int32_t)idx_pos : (int32_t)(own - span.first + span.lead + 1u);
        const int32_t lo = a.c.window && own + 1u > a.c.window + span.first ? (int32_t)(span.lead + own + 1u - a.c.window - span.first) : (int32_t)span.lead;
        const int32_t always = min((int32_t)(a.c.window ? max(a.c.sinks, span.lead) : span.lead), hi);
        const uint32_t *seen = a.visible ? a.visible + (uint64_t)token * words : nullptr;
        const uint32_t tm_s = tmem + s * 128u + ((warp & 3u) << 21), tm_o = tmem + 256u + s * 128u + ((warp & 3u) << 21);
        const int32_t lo_all = __reduce_max_sync(0xffffffffu, row_ok ? lo : 0), hi_all = __reduce_min_sync(0xffffffffu, row_ok ? hi : 0x7FFFFFFF);
        float m = -INFINITY, l = 0.f;
        for (uint32_t i = 0; i < my_n && alive; i++) {
            const int32_t key0 = (int32_t)((tile0 + (solo ? 2u * i + s : i)) * kManyKeys);
            /* what of the tile the row sees; a warp whose rows see it whole does without */
            const bool whole = key0 >= lo_all && key0 + (int32_t)kManyKeys <= hi_all;
            uint32_t vis[4] = {0u, 0u, 0u, 0u};
            if (!whole) {
#pragma unroll
                for (uint32_t ch = 0; ch < 4u; ch++) {
                    const int32_t k0 = key0 + (int32_t)(ch * 32u);
                    vis[ch] = bit_range(lo - k0, hi - k0) | bit_range(0 - k0, always - k0);
                    if (seen) {
                        const int32_t d = k0 - (int32_t)idx_pos;                         /* draft of the chunk's first key */
                        if (d > -32 && d < (int32_t)a.T) {
                            const uint32_t w0 = d >= 0 ? (uint32_t)d >> 5 : 0u, lo_word = seen[w0], hi_word = d >= 0 && w0 + 1u < words ? seen[w0 + 1u] : 0u;
                            vis[ch] |= (d >= 0 ? __funnelshift_r(lo_word, hi_word, (uint32_t)d & 31u) : lo_word << (uint32_t)(-d)) & bit_range(-d, (int32_t)a.T - d);
                        }
                    }
                }
            }
            alive = mbar_wait(s_full + s * 8u, i & 1u);
            if (!alive) break;
            tm_fence_after();
            if (whole) weights<true>(a.scale, tm_s, tm_o, HD, i != 0u, vis, m, l);
            else weights<false>(a.scale, tm_s, tm_o, HD, i != 0u, vis, m, l);
            tm_wait_store();
            tm_fence_before();
            arrive_warp(p_full + s * 8u);
        }
        uint32_t v[32];
        /* O, then the row's share or result */
        if (alive && my_n) { alive = mbar_wait(o_full + s * 8u, 0u); tm_fence_after(); }
        if (solo) {
            /* the second stream's share through shared memory (Q, K and V are done with: O1 is complete and O0 is awaited) */
            float *there = reinterpret_cast<float *>(many_raw + (base - smem_addr(many_raw)));
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (s == 1) {
                if (alive && my_n) {
#pragma unroll
                    for (uint32_t ch = 0; ch < HD / 32u; ch++) {
                        tm_load32(tm_o + ch * 32u, v);
                        tm_wait_load(); tm_hold(v);
#pragma unroll
                        for (uint32_t e = 0; e < 32u; e++) there[(ch * 32u + e) * 128u + wt] = __uint_as_float(v[e]);
                    }
                }
                there[HD * 128u + wt] = my_n ? m : -INFINITY; there[HD * 128u + 128u + wt] = l;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        if (alive && pos_ok && !(solo && s)) {
            const float *there = reinterpret_cast<const float *>(many_raw + (base - smem_addr(many_raw)));
            float f0 = 1.f, f1 = 0.f, total = l, top = m;
            if (solo) {
                const float m1 = there[HD * 128u + wt];
                top = fmaxf(m, m1);
                f0 = m == -INFINITY ? 0.f : exp2_fast(m - top); f1 = m1 == -INFINITY ? 0.f : exp2_fast(m1 - top);
                total = l * f0 + there[HD * 128u + 128u + wt] * f1;
            }
            const float r = total == 0.f ? 0.f : 1.f / total;
            /* (Q's place: this stream's products with it are done; solo: the ring's, where every product is, behind the second stream's share) */
            const uint32_t staged = base + (solo ? F::kRing + 8192u : F::kQ + s * F::kTile) + (warp & 3u) * 32u * HD * 2u;
            /* a share's outputs four dimensions at a time, rows side by side: what a warp writes (and the join reads) is one piece */
            const uint64_t block = ((uint64_t)split * gridDim.x + unit) * 2u + s;
            float *part = a.splits > 1u ? a.part_o + block * kManyRows * HD + wt * 4u : nullptr;
            if (a.splits > 1u && row_ok) *reinterpret_cast<float2 *>(a.part_ml + (block * kManyRows + wt) * 2u) = make_float2(!n ? -INFINITY : total == total ? top : 0.f /* a query that is not a number has no maximum, but its share counts */, total);
#pragma unroll
            for (uint32_t ch = 0; ch < HD / 32u; ch++) {
                if (my_n) { tm_load32(tm_o + ch * 32u, v); tm_wait_load(); tm_hold(v); }
                else {
#pragma unroll
                    for (uint32_t e = 0; e < 32u; e++) v[e] = 0u;
                }
                if (solo) {
#pragma unroll
                    for (uint32_t e = 0; e < 32u; e++) {
                        float x = __uint_as_float(v[e]) * f0;
                        if (f1 != 0.f) x = fmaf(there[(ch * 32u + e) * 128u + wt], f1, x);
                        v[e] = __float_as_uint(x);
                    }
                }
                if (row_ok && part) {
#pragma unroll
                    for (uint32_t e = 0; e < 32u; e += 4u) *reinterpret_cast<uint4 *>(part + (uint64_t)(ch * 8u + e / 4u) * kManyRows * 4u) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                } else if (!part) {
#pragma unroll
                    for (uint32_t e = 0; e < 32u; e += 8u) {
                        uint32_t w[4];
#pragma unroll
                        for (uint32_t j = 0; j < 4u; j++) w[j] = total == 0.f ? 0u : pack_bf16(__uint_as_float(v[e + 2u * j]) * r, __uint_as_float(v[e + 2u * j + 1u]) * r);
                        sts128u(staged + lane * (HD * 2u) + (((ch * 4u + e / 8u) ^ (lane & 7u)) << 4), w[0], w[1], w[2], w[3]);
                    }
                }
                __syncwarp();
            }
            if (!part) {
                /* the warp's 32 rows through shared memory, so that a store is whole rows */
                constexpr uint32_t kPieces = HD / 8u, kRowsOnce = 32u / kPieces;
#pragma unroll 4
                for (uint32_t r0 = 0; r0 < 32u; r0 += kRowsOnce) {
                    const uint32_t rr = r0 + lane / kPieces, piece = lane % kPieces, there_row = my_row0 + (warp & 3u) * 32u + rr;
                    const uint4 w = lds128(staged + rr * (HD * 2u) + ((piece ^ (rr & 7u)) << 4));
                    if (there_row < rows) *reinterpret_cast<uint4 *>(a.out + ((uint64_t)(there_row / group) * a.n_q + kvh * group + there_row % group) * HD + piece * 8u) = w;
                }
            }
        }
    } else if (warp < F::kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::kRegsProduce));
        /* ---- K and V into shared memory ---- */
        const uint32_t pt = tid - 256u, items = 2u * n;
        constexpr uint32_t kRowBytes = HD * (ELEM == kKvE4m3 ? 1u : 2u), kChunks = kRowBytes / 16u, kPasses = kManyKeys * kChunks / kProducers, kRowsPerPass = kProducers / kChunks;
        static_assert(kRowsPerPass % 8u == 0u, "a thread's rows take the same place in the swizzle");
        const uint32_t ch = pt % kChunks, r0 = pt / kChunks;                            /* this thread's chunk of rows r0, r0 + kRowsPerPass, ... */
        const uint64_t head = (uint64_t)kvh * a.c.capacity;
        auto tile_of = [&](uint32_t x) { return x == 0u ? 0u : x + 1u == items ? n - 1u : x & 1u ? (x + 1u) / 2u : (x - 2u) / 2u; };
        auto is_v = [&](uint32_t x) { return x != 0u && (x + 1u == items || !(x & 1u)); };
        auto slot_of = [&](uint32_t i) -> uint32_t {                                    /* of list index i < span.count */
            const uint32_t sl = i < span.lead ? i : slot_first + (i - span.lead);
            return i >= span.lead && sl >= a.c.capacity ? sl - ring : sl;
        };
        /* a tile of 128 keys whose slots follow one another needs one address */
        auto straight = [&](uint32_t i0) { return i0 + kManyKeys <= span.count && slot_of(i0 + kManyKeys - 1u) == slot_of(i0) + kManyKeys - 1u && (i0 >= span.lead || i0 + kManyKeys <= span.lead); };
        if constexpr (ELEM == kKvBf16) {
            /* a straight tile is one tensor-map copy per 64 dimensions (one thread, no multicast), any other is copied row by row */
            const uint32_t place = base + F::kRing + (ch >> 3) * F::kHalfBytes + swizzled(r0, ch & 7u), plane = a.layer * a.c.n_kv + kvh;
            uint32_t x = 0;
            for (; x < items && alive; x++) {
                const uint32_t i0 = (tile0 + tile_of(x)) * kManyKeys, to = base + F::kRing + (x % NS) * F::kTile, bar = full + (x % NS) * 8u;
                if (x >= NS) alive = mbar_wait(empty + (x % NS) * 8u, ((x / NS) - 1u) & 1u);
                if (!alive) break;
                if (straight(i0)) {
                    if (warp == 8u && lane == 0) {
                        mbar_expect(bar, F::kTile);
#pragma unroll
                        for (uint32_t h = 0; h < HD / 64u; h++) tensor_load(to + h * F::kHalfBytes, is_v(x) ? &vmap : &kmap, h * 64u, slot_of(i0), plane, bar);
                    }
                    __syncwarp();
                    if (warp != 8u) arrive_warp(bar);
                    continue;
                }
                const uint8_t *from = (is_v(x) ? a.c.v : a.c.k) + ch * 16u;
#pragma unroll
                for (uint32_t e = 0; e < kPasses; e++) {
                    const uint32_t i = i0 + r0 + e * kRowsPerPass;
                    copy16(place + (x % NS) * F::kTile + e * kRowsPerPass * 128u, from + (head + (i < span.count ? slot_of(i) : 0u)) * kRowBytes, i < span.count ? 16u : 0u);
                }
                copies_wait_all();
                async_proxy_fence();
                arrive_warp(bar);
            }
            /* Where the products gave up, copies may still be on their way: the CTA does not end before those of the last NS tiles
               have arrived (elsewhere they long have). */
            if (warp == 8u) for (uint32_t y = x > NS ? x - NS : 0u; y < x; y++) mbar_wait(full + (y % NS) * 8u, (y / NS) & 1u);
        } else {
            /* codes in registers a tile early (two sets, used in turn), widened into the operand's places */
            const uint32_t c8 = (ch & 3u) * 2u, place = base + F::kRing + (ch >> 2) * F::kHalfBytes, place_lo = place + swizzled(r0, c8), place_hi = place + swizzled(r0, c8 + 1u);
            auto load = [&](uint32_t x, uint4 (&w)[kPasses], uint8_t (&unit)[kPasses]) {
                if (x >= items) return;
                const bool v = is_v(x);
                const uint8_t *from = (v ? a.c.v : a.c.k) + ch * 16u, *exps = v ? a.c.v_exp : a.c.k_exp;
                const uint32_t i0 = (tile0 + tile_of(x)) * kManyKeys;
                if (straight(i0)) {
                    const uint64_t cell = head + slot_of(i0) + r0;
                    from += cell * kRowBytes; exps += cell;
#pragma unroll
                    for (uint32_t e = 0; e < kPasses; e++) { w[e] = *reinterpret_cast<const uint4 *>(from + e * kRowsPerPass * kRowBytes); unit[e] = exps[e * kRowsPerPass]; }
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < kPasses; e++) {
                        const uint32_t i = i0 + r0 + e * kRowsPerPass;
                        w[e] = make_uint4(0u, 0u, 0u, 0u); unit[e] = 0;
                        if (i < span.count) { const uint64_t cell = head + slot_of(i); w[e] = *reinterpret_cast<const uint4 *>(from + cell * kRowBytes); unit[e] = exps[cell]; }
                    }
                }
            };
            auto widen = [&](uint32_t x, const uint4 (&w)[kPasses], const uint8_t (&unit)[kPasses]) {
                if (x >= NS) alive = mbar_wait(empty + (x % NS) * 8u, ((x / NS) - 1u) & 1u);
                if (!alive) return;
                const uint32_t to = (x % NS) * F::kTile;
                bool large = false;
#pragma unroll
                for (uint32_t e = 0; e < kPasses; e++) large = large || unit[e] > 134u;
                large = __any_sync(0xffffffffu, large);
#pragma unroll
                for (uint32_t e = 0; e < kPasses; e++) {
                    /* code bits in bf16's places are the value times 2^-120: times 2^(120 + e), one exact multiplication while
                       that is a bf16 number (rows below 2^16), two beyond */
                    const uint32_t b = unit[e], f = min(b + 120u, 254u) * 0x00800080u, u[4] = {w[e].x, w[e].y, w[e].z, w[e].w};
                    uint32_t y[8];
#pragma unroll
                    for (uint32_t j = 0; j < 4u; j++) {
                        kv_spread(u[j], y[2 * j], y[2 * j + 1]);
                        y[2 * j] = kv_mul2(y[2 * j], f); y[2 * j + 1] = kv_mul2(y[2 * j + 1], f);
                    }
                    if (large) {
                        const uint32_t f2 = (max(b, 134u) - 7u) * 0x00800080u;
#pragma unroll
                        for (uint32_t j = 0; j < 8u; j++) y[j] = kv_mul2(y[j], f2);
                    }
                    sts128u(place_lo + to + e * kRowsPerPass * 128u, y[0], y[1], y[2], y[3]);
                    sts128u(place_hi + to + e * kRowsPerPass * 128u, y[4], y[5], y[6], y[7]);
                }
                async_proxy_fence();
                arrive_warp(full + (x % NS) * 8u);
            };
            uint4 w0[kPasses], w1[kPasses];
            uint8_t u0[kPasses], u1[kPasses];
            load(0u, w0, u0);
            for (uint32_t x = 0; x < items && alive; x += 2u) {                         /* (the number of items is even) */
                load(x + 1u, w1, u1);
                widen(x, w0, u0);
                if (!alive) break;
                load(x + 2u, w0, u0);
                widen(x + 1u, w1, u1);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::kRegsMma));
        if (warp == F::kMmaWarp && n) {
            /* ---- matrix products ---- */
            constexpr uint32_t kIdescS = idesc_bf16(128u, kManyKeys, false), kIdescO = idesc_bf16(128u, HD, true);
            const uint32_t leader = elect_lane();
            /* descriptors of Q and of the ring's first slot, as a row-major (K) and as a transposed operand (V); the address field counts 16 bytes */
            const uint32_t q_desc = desc_low(base + F::kQ, 16u), k_desc = desc_low(base + F::kRing, 16u), v_desc = desc_low(base + F::kRing, F::kHalfBytes);
            auto ready = [&](uint32_t item) { return mbar_wait(full + (item % NS) * 8u, (item / NS) & 1u); };
            auto scores = [&](uint32_t s, uint32_t t) {
                const uint32_t qd = q_desc + (solo ? 0u : s * (F::kTile >> 4)), kd = k_desc + (item_k(t) % NS) * (F::kTile >> 4);
#pragma unroll
                for (uint32_t kk = 0; kk < HD / 16u; kk++) {
                    constexpr uint32_t kHalf = F::kHalfBytes >> 4;
                    mma_ss(leader, tmem + s * 128u, qd + (kk >> 2) * kHalf + (kk & 3u) * 2u, kd + (kk >> 2) * kHalf + (kk & 3u) * 2u, kIdescS, kk ? 1u : 0u);
                }
                mma_commit(leader, s_full + s * 8u);
            };
            auto outputs = [&](uint32_t s, uint32_t t, bool first) {
                const uint32_t vd = v_desc + (item_v(t) % NS) * (F::kTile >> 4);
#pragma unroll
                for (uint32_t kk = 0; kk < kManyKeys / 16u; kk++)
                    mma_ts(leader, tmem + 256u + s * 128u, tmem + s * 128u + kk * 8u, vd + kk * (2048u >> 4), kIdescO, first && !kk ? 0u : 1u);
            };
            auto release = [&](uint32_t item) { mma_commit(leader, empty + (item % NS) * 8u); };
            /* step x = one stream's tile: S of the first tile of each, then per step O += P V and the S that follows it.  Alone
               (solo), tile x belongs to stream x & 1; together, both streams take tile x / 2. */
            const uint32_t steps = solo ? n : 2u * n;
            alive = mbar_wait(q_full, 0u) && (solo || mbar_wait(q_full + 8u, 0u));
            for (uint32_t x = 0; x < steps + 2u && alive; x++) {
                const uint32_t s = x & 1u;
                if (x >= 2u) {
                    const uint32_t y = x - 2u, t = solo ? y : y >> 1;
                    alive = ready(item_v(t)) && mbar_wait(p_full + s * 8u, (y >> 1) & 1u);
                    if (!alive) break;
                    tm_fence_after();
                    outputs(s, t, y < 2u);
                    if (solo || s) release(item_v(t));
                    if (x >= steps) mma_commit(leader, o_full + s * 8u);
                }
                if (x < steps) {
                    const uint32_t t = solo ? x : x >> 1;
                    alive = ready(item_k(t));
                    if (!alive) break;
                    tm_fence_after();
                    scores(s, t);
                    if (solo || s) release(item_k(t));
                }
            }
            if (!alive) {                                                               /* what was issued must end before the memory is given back */
                mma_commit(leader, o_full); mma_commit(leader, o_full + 8u);
                for (uint32_t i = 0; i < (1u << 20); i++) if (__all_sync(0xffffffffu, mbar_poll(o_full, 0u) && mbar_poll(o_full + 8u, 0u))) break;
            }
        }
    }
    if (!pos_ok && tid == 0) atomicOr(a.status, kKvStatusPosition);
    report_wait(alive, a.status);
    __syncwarp();
    tm_fence_before();
    __syncthreads();
    tm_fence_after();
    if (warp == F::kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

/* The shares of the splits joined, in their order.  A lane is a row, a warp 32 rows and 16 dimensions of them; `ways` warps take
   the splits in turn and meet in shared memory. */
template <int HD>
__global__ void __launch_bounds__(256) kv_attention_many_join_kernel(const KvAttention a, uint32_t units, uint32_t ways) {
    constexpr uint32_t kPieces = HD / 16u;
    __shared__ float sums[8][17][32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, way = warp % ways;
    const uint64_t item = (uint64_t)blockIdx.x * (8u / ways) + warp / ways;             /* unit, stream, 32 rows, 16 dimensions */
    const uint32_t piece = (uint32_t)(item % kPieces), part = (uint32_t)(item / kPieces) & 3u, s = (uint32_t)(item / (kPieces * 4u)) & 1u;
    const uint64_t unit = item / (kPieces * 8u);
    kv_dependency_sync();
    const int32_t pos = *a.pos;
    if (pos < 0 || (uint64_t)pos + a.T > (a.c.window ? 0x7FFFFFFFu : a.c.capacity)) return;
    const uint32_t group = a.n_q / a.c.n_kv, rows = a.T * group, kvh = (uint32_t)(unit % a.c.n_kv), row0 = (uint32_t)(unit / a.c.n_kv) * 2u * kManyRows, r = part * 32u + lane, row = row0 + s * kManyRows + r;
    const bool here = unit < units && row0 < rows && !(s && rows - row0 <= kManyRows), live = here && row < rows;      /* (a unit of one row tile: the streams' shares are one) */
    float top = -INFINITY, total = 0.f, sum[16];
#pragma unroll
    for (uint32_t j = 0; j < 16u; j++) sum[j] = 0.f;
    if (live) {
        const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + (unit * 2u + s) * kManyRows + r;
        const float4 *from = reinterpret_cast<const float4 *>(a.part_o) + (unit * 2u + s) * kManyRows * (HD / 4u) + (uint64_t)piece * 4u * kManyRows + r;
        const uint64_t step = (uint64_t)units * 2u * kManyRows;                         /* from split to split */
#pragma unroll 4
        for (uint32_t y = 0; y < a.splits; y++) top = fmaxf(top, __ldcg(ml + y * step).x);
#pragma unroll 2
        for (uint32_t y = way; y < a.splits; y += ways) {
            const float2 w = __ldcg(ml + y * step);
            float4 v[4];
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++) v[j] = __ldcg(from + y * step * (HD / 4u) + j * kManyRows);
            const bool share = w.x != -INFINITY;                                        /* (one without keys left no outputs) */
            const float f = share ? exp2_fast(w.x - top) : 0.f;
            total = fmaf(w.y, f, total);
            if (share) {
#pragma unroll
                for (uint32_t j = 0; j < 4u; j++) {
                    sum[4 * j] = fmaf(v[j].x, f, sum[4 * j]); sum[4 * j + 1] = fmaf(v[j].y, f, sum[4 * j + 1]);
                    sum[4 * j + 2] = fmaf(v[j].z, f, sum[4 * j + 2]); sum[4 * j + 3] = fmaf(v[j].w, f, sum[4 * j + 3]);
                }
            }
        }
    }
    if (ways > 1u) {
#pragma unroll
        for (uint32_t j = 0; j < 16u; j++) sums[warp][j][lane] = sum[j];
        sums[warp][16][lane] = total;
        __syncthreads();
        if (way) return;
        for (uint32_t w = 1; w < ways; w++) {
            total += sums[warp + w][16][lane];
#pragma unroll
            for (uint32_t j = 0; j < 16u; j++) sum[j] += sums[warp + w][j][lane];
        }
    }
    if (!live) return;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    uint4 *to = reinterpret_cast<uint4 *>(a.out + ((uint64_t)(row / group) * a.n_q + kvh * group + row % group) * HD + piece * 16u);
#pragma unroll
    for (uint32_t j = 0; j < 2u; j++)
        to[j] = make_uint4(pack_bf16(sum[8 * j] * inv, sum[8 * j + 1] * inv), pack_bf16(sum[8 * j + 2] * inv, sum[8 * j + 3] * inv),
                           pack_bf16(sum[8 * j + 4] * inv, sum[8 * j + 5] * inv), pack_bf16(sum[8 * j + 6] * inv, sum[8 * j + 7] * inv));
}

/* cuTensorMapEncodeTiled through the runtime's driver entry point (the library does not link against the driver) */
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_tiled() {
    static std::atomic<void *> cached{nullptr};
    void *fn = cached.load(std::memory_order_acquire);
    if (!fn) {
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &res) != cudaSuccess || res != cudaDriverEntryPointSuccess) { cudaGetLastError(); return nullptr; }
        cached.store(fn, std::memory_order_release);
    }
    return reinterpret_cast<EncodeTiledFn>(fn);
}

template <int HD, int ELEM>
static cudaError_t launch_many(cudaStream_t st, const KvAttention &given, int sms) {
    /* Units of one key/value head's 256 rows, one CTA each (times the splits of the keys).  Where the last wave of CTAs would fill
       less than half of the GPU, its rows go out as units of 128: twice as many, each done in half the time (its two streams
       take the key tiles in turn).  4096 tokens of 32 + 8 heads under a window of 4096, 512 units: 308 us (sustained), with halved ones 292. */
    const uint64_t rows = (uint64_t)given.T * (given.n_q / given.c.n_kv), all = (rows + 2u * kManyRows - 1u) / (2u * kManyRows) * given.c.n_kv, last = all % (uint64_t)sms;
    KvAttention a = given;
    uint64_t units = all;
    a.pairs = (uint32_t)all;
    if (a.splits == 1u && all > (uint64_t)sms && last && last * 2u <= (uint64_t)sms) {
        const uint64_t halved = (last + given.c.n_kv - 1u) / given.c.n_kv;              /* pairs of row tiles of every head */
        if (halved * given.c.n_kv * 2u <= (uint64_t)sms) {
            const uint64_t kept = all / given.c.n_kv - halved, left = rows - kept * 2u * kManyRows;
            a.pairs = (uint32_t)(kept * given.c.n_kv); units = a.pairs + (left + kManyRows - 1u) / kManyRows * given.c.n_kv;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((uint32_t)units, a.splits); cfg.blockDim = dim3(Many<HD, ELEM>::kThreads); cfg.dynamicSmemBytes = Many<HD, ELEM>::kSmem; cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = dependent_launch() ? 1 : 0;
    /* bf16: K and V as [planes][capacity][HD], boxes of 64 dimensions x 128 rows, swizzled as the operands are */
    alignas(64) CUtensorMap maps[2] = {};
    if (ELEM == kKvBf16) {
        const EncodeTiledFn encode = encode_tiled();
        if (!encode) return cudaErrorNotSupported;
        const cuuint64_t dims[3] = {HD, a.c.capacity, (cuuint64_t)a.layers * a.c.n_kv}, strides[2] = {HD * 2u, (cuuint64_t)a.c.capacity * HD * 2u};
        const cuuint32_t box[3] = {64u, kManyKeys, 1u}, ones[3] = {1u, 1u, 1u};
        const uint64_t below = (uint64_t)a.layer * a.c.n_kv * a.c.capacity * HD * 2u;
        for (int i = 0; i < 2; i++)
            if (encode(&maps[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3u, (i ? a.c.v : a.c.k) - below, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) return cudaErrorInvalidValue;
    }
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kv_attention_many_kernel<HD, ELEM>, a, maps[0], maps[1]);
    if (err != cudaSuccess || a.splits == 1u) return err;
    const uint32_t ways = a.splits >= 16u ? 8u : a.splits >= 6u ? 4u : a.splits >= 3u ? 2u : 1u;
    cfg.gridDim = dim3((uint32_t)((units * 8u * (HD / 16u) * ways + 7u) / 8u)); cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;                                                                   /* (its set-up overlaps the last CTAs; it waits for the whole grid before it reads) */
    return cudaLaunchKernelEx(&cfg, kv_attention_many_join_kernel<HD>, a, (uint32_t)units, ways);
}

cudaError_t launch_kv_many(cudaStream_t st, int elem, uint32_t head_dim, const KvAttention &a, int sms) {
    if (elem == kKvE4m3) return head_dim == 64u ? launch_many<64, kKvE4m3>(st, a, sms) : launch_many<128, kKvE4m3>(st, a, sms);
    return head_dim == 64u ? launch_many<64, kKvBf16>(st, a, sms) : launch_many<128, kKvBf16>(st, a, sms);
}

/* One warp waits, with a short limit, for a barrier that nothing arrives at, and reports it as the attention does. */
__global__ void kv_wait_probe_kernel(int *status) {
    __shared__ __align__(8) uint64_t bar;
    if (threadIdx.x == 0) { mbar_init(smem_addr(&bar), 1u); mbar_init_fence(); }
    __syncwarp();
    report_wait(mbar_wait(smem_addr(&bar), 0u, 64u), status);
}
cudaError_t launch_kv_wait_probe(cudaStream_t st, int *status) {
    kv_wait_probe_kernel<<<1, 32, 0, st>>>(status);
    return cudaGetLastError();
}

void configure_kv_many() {
    cudaFuncSetAttribute(kv_attention_many_kernel<64, kKvBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Many<64, kKvBf16>::kSmem);
    cudaFuncSetAttribute(kv_attention_many_kernel<64, kKvE4m3>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Many<64, kKvE4m3>::kSmem);
    cudaFuncSetAttribute(kv_attention_many_kernel<128, kKvBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Many<128, kKvBf16>::kSmem);
    cudaFuncSetAttribute(kv_attention_many_kernel<128, kKvE4m3>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Many<128, kKvE4m3>::kSmem);
}

int read_kv_status(bool clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_kernel_status, sizeof(int)) != cudaSuccess) return -1;
    if (clear && v) { const int z = 0; cudaMemcpyToSymbol(g_kernel_status, &z, sizeof(int)); }
    return v;
}

}  // namespace nwc
