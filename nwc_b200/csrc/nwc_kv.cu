/* The cache that is quantised as it is written: store (per-head RMSNorm, rotary positions, rounding to the cache's type),
 * read back, and the move of an accepted draft path.  Formats and slot rules: nwc_kv.h.
 *
 * All three move bytes: their floor is the bytes in and out at the memory's rate, and for one token a launch.
 */
#include <cuda_fp8.h>
#include "nwc_kv.h"
#include "nwc_launch.h"

#define NWC_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

using namespace nwc;

__device__ __forceinline__ void dependency_sync() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ float lo16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi16(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { uint32_t d; asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a)); return d; }
__device__ __forceinline__ uint16_t pack_e4m3(float a, float b) { return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3); }

__device__ __forceinline__ uint4 pack8(const float (&y)[8]) { return make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7])); }
constexpr float kLargestBf16 = 3.3895313892515355e38f;
/* 1.875 * 2^127: the largest value of three mantissa bits in range; rounding a larger one up would reach 2^128 */
constexpr float kLargestE4m3 = 3.1901471898837980e38f;
/* a + b as the rounded sum and what the rounding left (Knuth's two-sum) */
__device__ __forceinline__ float two_sum(float a, float b, float &e) {
    const float s = __fadd_rn(a, b), t = __fsub_rn(s, a);
    e = __fadd_rn(__fsub_rn(a, __fsub_rn(s, t)), __fsub_rn(b, t));
    return s;
}
/* exponent byte of a row: smallest e with top <= 1.75 * 2^(8 + e), from top's exponent field, one more where its mantissa is above 0.75 */
__device__ __forceinline__ int32_t unit_byte(float top) {
    const uint32_t bits = __float_as_uint(top);
    return max(0, (int32_t)(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0));
}

struct StoreArgs {
    KvLayer c;
    const uint16_t *qkv; uint64_t ldqkv;
    uint32_t T, n_q;
    const uint16_t *q_norm, *k_norm, *cos_t, *sin_t;
    uint32_t max_pos;
    const int32_t *pos, *depth;
    float eps;
    uint16_t *q_out;
    int *status;
    uint32_t chunks;             /* kStoreQ passes of query rows that a warp takes one after the other */
};

/* HD / 8 lanes hold one row, eight numbers each: four of the lower half and the four that rotary embedding pairs them with, so a
   row is two 8-byte loads per lane and no number has to be fetched from another lane (41 us with shuffles, 39 without, for the
   call below).  A warp takes PASSES x kSide rows of one kind (query, key or value) of one token: their loads are in
   flight together, before the position is known, and they share the token's cos / sin.  (Rows of all kinds in one warp make
   one long piece of code, four times unrolled: 100 us for 4096 tokens of 64 + 16 heads where this takes a third, most of it waiting
   for instructions.)
   Between the loaded bf16 numbers and what is stored is fp32, rounded once.  Keys that become e4m3 codes are kept to twice
   fp32's precision on the way (with fp32's few roundings some four of a million land on the wrong side of a code's border):
   a product of three bf16 numbers is exact in fp32, so x w cos and x' w' sin are, their sum is two numbers, and so is the
   reciprocal norm after one Newton step. */
template <int HD> struct Row {
    static constexpr uint32_t kLanes = HD / 8, kSide = 32 / kLanes;
    static __device__ __forceinline__ float sum(float v) {
#pragma unroll
        for (uint32_t o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    static __device__ __forceinline__ float max(float v) {
#pragma unroll
        for (uint32_t o = kLanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    }
};
__device__ __forceinline__ void unpack8(const uint4 &w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; j++) { x[2 * j] = lo16(u[j]); x[2 * j + 1] = hi16(u[j]); }
}
/* a lane's eight numbers of a row: 4 sub .. 4 sub + 3 and the same of the upper half */
template <int HD> __device__ __forceinline__ uint4 load_streamed(const uint16_t *row) {
    const uint2 a = __ldcs(reinterpret_cast<const uint2 *>(row)), b = __ldcs(reinterpret_cast<const uint2 *>(row + HD / 2));
    return make_uint4(a.x, a.y, b.x, b.y);
}
template <int HD> __device__ __forceinline__ uint4 load_again(const uint16_t *row) {
    const uint2 a = *reinterpret_cast<const uint2 *>(row), b = *reinterpret_cast<const uint2 *>(row + HD / 2);
    return make_uint4(a.x, a.y, b.x, b.y);
}
template <int HD> __device__ __forceinline__ void store_halves(uint16_t *row, const uint4 &w) {
    *reinterpret_cast<uint2 *>(row) = make_uint2(w.x, w.y); *reinterpret_cast<uint2 *>(row + HD / 2) = make_uint2(w.z, w.w);
}
/* x w / norm, turned (s: with the sign of the partner's share) */
template <int HD>
__device__ __forceinline__ void normed_and_turned(float (&y)[8], bool norm, const float (&w)[8], float eps, const float (&c)[8], const float (&s)[8]) {
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) ss = fmaf(y[j], y[j], ss);
        const float inv = rsqrtf(Row<HD>::sum(ss) * (1.f / HD) + eps);
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] *= inv * w[j];
    }
#pragma unroll
    for (int j = 0; j < 4; j++) { const float a = y[j], b = y[j + 4]; y[j] = fmaf(a, c[j], b * s[j]); y[j + 4] = fmaf(b, c[j + 4], a * s[j + 4]); }
}
/* the same as a sum of two numbers each */
template <int HD>
__device__ __forceinline__ void normed_and_turned_exactly(float (&y)[8], float (&low)[8], bool norm, const float (&w)[8], float eps, const float (&c)[8], const float (&s)[8]) {
    float inv = 1.f, inv_low = 0.f;
    if (norm) {
        float sh = 0.f, sl = 0.f, e;
#pragma unroll
        for (int j = 0; j < 8; j++) { sh = two_sum(sh, y[j] * y[j], e); sl += e; }
#pragma unroll
        for (uint32_t o = Row<HD>::kLanes / 2; o > 0; o >>= 1) {
            const float oh = __shfl_xor_sync(0xffffffffu, sh, o), ol = __shfl_xor_sync(0xffffffffu, sl, o);
            sh = two_sum(sh, oh, e); sl = sl + ol + e;
        }
        const float mh = two_sum(sh * (1.f / HD), eps, e), ml = sl * (1.f / HD) + e;
        inv = rsqrtf(mh);
        const float ph = __fmul_rn(inv, inv), pl = fmaf(inv, inv, -ph);
        inv_low = 0.5f * inv * (fmaf(-mh, ph, 1.f) - fmaf(mh, pl, ml * ph));
    }
    float xw[8];
#pragma unroll
    for (int j = 0; j < 8; j++) xw[j] = norm ? __fmul_rn(y[j], w[j]) : y[j];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float e, h = two_sum(__fmul_rn(xw[j], c[j]), __fmul_rn(xw[j ^ 4], s[j]), e);
        if (norm) {
            const float p = __fmul_rn(h, inv), q = fmaf(h, inv, -p) + fmaf(e, inv, h * inv_low);
            h = __fadd_rn(p, q); e = __fsub_rn(q, __fsub_rn(h, p));
        }
        y[j] = h; low[j] = e;
    }
}
/* One row's eight numbers y + low of this lane into the cache.  What is not finite would reach every query: it is kept out (0)
   and reported. */
template <int HD, int ELEM>
__device__ __forceinline__ void store_row(const StoreArgs &a, uint8_t *plane, uint8_t *exps, uint64_t cell, uint32_t sub, bool live, float (&y)[8], float (&low)[8]) {
    bool fine = true;
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if (!(fabsf(y[j]) <= kLargestBf16)) { fine = false; y[j] = low[j] = 0.f; }
        if (ELEM == kKvE4m3) {
            if (fabsf(y[j]) >= kLargestE4m3) { y[j] = copysignf(kLargestE4m3, y[j]); low[j] = 0.f; }
            /* the magnitude rounded up: what the row's unit goes by */
            top = fmaxf(top, __uint_as_float(__float_as_uint(fabsf(y[j])) + (low[j] != 0.f && (low[j] > 0.f) == (y[j] > 0.f) ? 1u : 0u)));
        }
    }
    if (ELEM == kKvE4m3) {
        const int32_t b = unit_byte(Row<HD>::max(top));
        const float up = __uint_as_float((uint32_t)(254 - b) << 23);  /* 2^(127 - b): exact */
#pragma unroll
        for (int j = 0; j < 8; j++) {                                 /* truncated with a sticky last bit: rounding that to e4m3 is rounding the sum of both numbers */
            uint32_t f = __float_as_uint(y[j]);
            if (low[j] != 0.f) f = (f - ((low[j] > 0.f) == (y[j] > 0.f) ? 0u : 1u)) | 1u;
            y[j] = __uint_as_float(f) * up;
        }
        if (live) {
            *reinterpret_cast<uint32_t *>(plane + cell * HD + sub * 4u) = pack_e4m3(y[0], y[1]) | ((uint32_t)pack_e4m3(y[2], y[3]) << 16);
            *reinterpret_cast<uint32_t *>(plane + cell * HD + HD / 2 + sub * 4u) = pack_e4m3(y[4], y[5]) | ((uint32_t)pack_e4m3(y[6], y[7]) << 16);
            if (sub == 0) exps[cell] = (uint8_t)b;
        }
    } else if (live) store_halves<HD>(reinterpret_cast<uint16_t *>(plane) + cell * HD + sub * 4u, pack8(y));
    if (live && !fine) atomicOr(a.status, kKvStatusNotFinite);
}

constexpr uint32_t kStoreQ = 4, kStoreK = 1, kStoreV = 2;             /* passes of a warp */
template <int HD> __host__ __device__ constexpr uint32_t store_groups(uint32_t n, uint32_t passes) { return (n + passes * (256u / HD) - 1u) / (passes * (256u / HD)); }

/* Bound: latency.  A warp's life is short and its loads depend on one another (rows, position, cos / sin); 4096 tokens of 64 +
   16 heads without norms take 34 us for 160 MB, 0.73 of measured bandwidth, with 2.7 instructions of 4 per clock, the ALU at 55 % and waiting
   for memory the largest stall.  So the warps that fit count: without the norm weights the kernel is held to 64 registers (four
   CTAs per SM; with 80 and three it takes 39; two bf16 forms spill 8 bytes for it), with them it would spill more than it gains
   (one token 2.8 -> 3.3 us, 517 tokens 5.9 -> 7.1, 4096 tokens no faster). */
template <int HD, int ELEM, bool NORM>
__global__ void __launch_bounds__(256, NORM ? 3 : 4) kv_store_kernel(const StoreArgs a) {
    using R = Row<HD>;
    const uint32_t lane = threadIdx.x & 31u, sub = lane % R::kLanes, side = lane / R::kLanes, d0 = sub * 4u, n_q = a.n_q, n_kv = a.c.n_kv;
    const uint32_t gq = store_groups<HD>(n_q, kStoreQ * a.chunks), gk = store_groups<HD>(n_kv, kStoreK), gv = store_groups<HD>(n_kv, kStoreV), groups = gq + gk + gv;
    const uint32_t unit = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);           /* (below 2^31: the launcher checks) */
    dependency_sync();
    if (unit >= groups * a.T) return;
    const uint32_t t = unit / groups, group = unit - t * groups;
    const int kind = group < gq ? 0 : group < gq + gk ? 1 : 2;        /* of the whole warp */
    const uint32_t n = kind ? n_kv : n_q, row0 = kind == 0 ? group * a.chunks * kStoreQ * R::kSide : kind == 1 ? (group - gq) * kStoreK * R::kSide : (group - gq - gk) * kStoreV * R::kSide;
    const uint16_t *from = a.qkv + (uint64_t)t * a.ldqkv + (uint64_t)(kind == 0 ? 0u : kind == 1 ? n_q : n_q + n_kv) * HD + d0;
    uint4 raw[kStoreQ];
#pragma unroll
    for (uint32_t i = 0; i < kStoreQ; i++) {
        const uint32_t row = row0 + i * R::kSide + side;
        raw[i] = row < n && (i == 0u || kind == 0 || (kind == 2 && i < kStoreV)) ? load_streamed<HD>(from + (uint64_t)row * HD) : make_uint4(0u, 0u, 0u, 0u);
    }
    const int32_t pos = *a.pos, depth = a.depth ? a.depth[t] : (int32_t)t;
    const uint32_t limit = a.c.window ? 0x7FFFFFFFu : a.c.capacity;
    const bool ok = pos >= 0 && (uint64_t)pos + a.T <= limit && depth >= 0 && (uint32_t)depth < a.T && (uint64_t)pos + (a.depth ? (uint32_t)depth + 1u : a.T) <= a.max_pos;
    if (!ok) { if (lane == 0) atomicOr(a.status, kKvStatusPosition); return; }
    const uint64_t slot = kv_slot((uint32_t)pos + t, a.c.capacity, a.c.window, a.c.sinks);
    if (kind == 2) {
#pragma unroll
        for (uint32_t i = 0; i < kStoreV; i++) {
            const uint32_t row = row0 + i * R::kSide + side;
            float y[8], low[8];
            unpack8(raw[i], y);
#pragma unroll
            for (int j = 0; j < 8; j++) low[j] = 0.f;
            store_row<HD, ELEM>(a, a.c.v, a.c.v_exp, (uint64_t)row * a.c.capacity + slot, sub, row < n, y, low);
        }
        return;
    }
    const uint64_t at = ((uint64_t)pos + (uint32_t)depth) * HD + d0;
    float c[8], s[8], w[8];
    unpack8(load_again<HD>(a.cos_t + at), c);
    unpack8(load_again<HD>(a.sin_t + at), s);
    if (NORM) unpack8(load_again<HD>((kind ? a.k_norm : a.q_norm) + d0), w);
#pragma unroll
    for (int j = 0; j < 4; j++) s[j] = -s[j];                         /* the lower half takes the upper one's numbers negated */
    if (kind == 1) {
        static_assert(kStoreK == 1, "one pass of keys");
        const uint32_t row = row0 + side;
        float y[8], low[8];
        unpack8(raw[0], y);
        if (ELEM == kKvE4m3) normed_and_turned_exactly<HD>(y, low, NORM, w, a.eps, c, s);
        else normed_and_turned<HD>(y, NORM, w, a.eps, c, s);
        store_row<HD, ELEM>(a, a.c.k, a.c.k_exp, (uint64_t)row * a.c.capacity + slot, sub, row < n, y, low);
        return;
    }
    for (uint32_t chunk = 0; chunk < a.chunks; chunk++) {
        const uint32_t first = row0 + chunk * kStoreQ * R::kSide + side;
        uint4 next[kStoreQ];
#pragma unroll
        for (uint32_t i = 0; i < kStoreQ; i++) {
            const uint32_t row = first + (kStoreQ + i) * R::kSide;
            next[i] = chunk + 1u < a.chunks && row < n ? load_streamed<HD>(from + (uint64_t)row * HD) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (uint32_t i = 0; i < kStoreQ; i++) {
            const uint32_t row = first + i * R::kSide;
            float y[8];
            unpack8(raw[i], y);
            normed_and_turned<HD>(y, NORM, w, a.eps, c, s);
            if (row < n) store_halves<HD>(a.q_out + ((uint64_t)t * n_q + row) * HD + d0, pack8(y));
            raw[i] = next[i];
        }
    }
}

struct ReadArgs {
    KvLayer c;
    uint32_t first, count, head_dim;
    uint16_t *k_out, *v_out;     /* bf16 [n_kv][count][head_dim] */
};

/* One thread reads back 16 numbers; K (blockIdx.z = 0) and V (1) of one head per blockIdx.y. */
template <int ELEM>
__global__ void __launch_bounds__(256) kv_read_kernel(const ReadArgs a) {
    const uint32_t per_row = a.head_dim >> 4;
    const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    dependency_sync();
    if (i >= (uint64_t)a.count * per_row) return;
    const uint32_t r = (uint32_t)(i / per_row), d0 = (uint32_t)(i % per_row) * 16u;
    const uint64_t cell = (uint64_t)blockIdx.y * a.c.capacity + kv_slot(a.first + r, a.c.capacity, a.c.window, a.c.sinks);
    const uint8_t *from = blockIdx.z ? a.c.v : a.c.k;
    uint4 *to = reinterpret_cast<uint4 *>((blockIdx.z ? a.v_out : a.k_out) + ((uint64_t)blockIdx.y * a.count + r) * a.head_dim + d0);
    if (ELEM == kKvE4m3) {
        const uint4 w = *reinterpret_cast<const uint4 *>(from + cell * a.head_dim + d0);
        const uint32_t unit2 = kv_unit2((blockIdx.z ? a.c.v_exp : a.c.k_exp)[cell]);
        uint4 lo, hi;
        kv_values4(w.x, unit2, lo.x, lo.y); kv_values4(w.y, unit2, lo.z, lo.w);
        kv_values4(w.z, unit2, hi.x, hi.y); kv_values4(w.w, unit2, hi.z, hi.w);
        to[0] = lo; to[1] = hi;
    } else {
        const uint4 *src = reinterpret_cast<const uint4 *>(from + (cell * a.head_dim + d0) * 2u);
        const uint4 lo = src[0], hi = src[1];
        to[0] = lo; to[1] = hi;
    }
}

/* The accepted path of a draft tree, moved together: row pos + path[i] -> row pos + i for i < count, in every layer and head
   (one CTA each).  path rises strictly, so path[i] >= i: a row is never overwritten before the moves that read it, as long as
   the moves run in order or read before they write.  A CTA takes kMoves x 256 pieces of 16 bytes at a time, all read before
   any is written.  (One thread per piece's column, row after row: 5 us for 15 rows, a load's latency each, where this takes 3.) */
constexpr uint32_t kMoves = 4;
__global__ void __launch_bounds__(256) kv_commit_kernel(KvLayer c, uint32_t row_bytes, uint32_t T, const int32_t *pos_ptr, const int32_t *path, const int32_t *count_ptr, uint32_t most, int *status) {
    __shared__ uint32_t from[NWC_KV_MAX_TREE];                        /* slots */
    const uint32_t tid = threadIdx.x;
    dependency_sync();
    const int32_t pos = *pos_ptr, count = *count_ptr;
    const uint64_t end = c.window ? 0x7FFFFFFFu : c.capacity;
    bool ok = pos >= 0 && count >= 0 && (uint32_t)count <= most;
    if (ok) {
        for (uint32_t i = tid; i < (uint32_t)count; i += 256u) {
            const int32_t p = path[i], before = i ? path[i - 1u] : -1;
            ok = ok && p > before && (uint32_t)p < T && (uint64_t)pos + (uint32_t)p < end;
            from[i] = kv_slot((uint32_t)(pos + p), c.capacity, c.window, c.sinks);
        }
    }
    if (!__syncthreads_and(ok)) { if (tid == 0) atomicOr(status, kKvStatusPath); return; }
    const uint64_t cell0 = (uint64_t)blockIdx.x * c.capacity;
    const uint32_t columns = row_bytes >> 4, pieces = 2u * columns * (uint32_t)count;
    auto place = [&](uint32_t e, uint32_t slot) {                    /* piece e = row i, K's columns, V's columns */
        const uint32_t j = e % (2u * columns);
        return reinterpret_cast<uint4 *>((j < columns ? c.k : c.v) + (cell0 + slot) * row_bytes + (j % columns) * 16u);
    };
    auto target = [&](uint32_t i) { return kv_slot((uint32_t)pos + i, c.capacity, c.window, c.sinks); };
    for (uint32_t e0 = 0; e0 < pieces; e0 += kMoves * 256u) {
        uint4 w[kMoves];
#pragma unroll
        for (uint32_t m = 0; m < kMoves; m++) { const uint32_t e = e0 + m * 256u + tid; if (e < pieces) w[m] = *place(e, from[e / (2u * columns)]); }
        __syncthreads();
#pragma unroll
        for (uint32_t m = 0; m < kMoves; m++) { const uint32_t e = e0 + m * 256u + tid; if (e < pieces) *place(e, target(e / (2u * columns))) = w[m]; }
        __syncthreads();
    }
    for (uint32_t e0 = 0; c.k_exp && e0 < 2u * (uint32_t)count; e0 += 256u) {
        const uint32_t e = e0 + tid;
        uint8_t *exps = (e & 1u ? c.v_exp : c.k_exp) + cell0, w = 0;
        if (e < 2u * (uint32_t)count) w = exps[from[e >> 1]];
        __syncthreads();
        if (e < 2u * (uint32_t)count) exps[target(e >> 1)] = w;
        __syncthreads();
    }
}

template <class... Params, class... Args>
cudaError_t launch(void (*kernel)(Params...), dim3 grid, dim3 block, void *stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = nwc::dependent_launch() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

bool aligned16(const void *p) { return !(reinterpret_cast<uintptr_t>(p) & 15u); }

/* the cache is one the kernels can address, and T tokens at once fit beside what its window still has to see */
bool cache_ok(const nwc_kv_cache *c, uint32_t layer, uint32_t T) {
    if (!c || !c->layers || layer >= c->layers || !c->n_kv || !c->capacity || c->capacity > 0x7FFFFF00u || (c->elem != kKvBf16 && c->elem != kKvE4m3)) return false;
    if (c->head_dim != 64u && c->head_dim != 128u && c->head_dim != 256u) return false;
    if (!c->k || !c->v || !aligned16(c->k) || !aligned16(c->v) || (c->elem == kKvE4m3 && (!c->k_exp || !c->v_exp))) return false;
    if ((uint64_t)c->layers * c->n_kv > 0x7FFFFFFFull) return false;
    if (c->window) return c->sinks < c->capacity && (uint64_t)c->window + (T ? T - 1u : 0u) <= c->capacity - c->sinks;
    return T <= c->capacity;
}
KvLayer layer_of(const nwc_kv_cache *c, uint32_t layer) {
    const uint64_t cells = (uint64_t)layer * c->n_kv * c->capacity, bytes = cells * c->head_dim * (c->elem == kKvBf16 ? 2u : 1u);
    const bool q = c->elem == kKvE4m3;
    return KvLayer{static_cast<uint8_t *>(c->k) + bytes, static_cast<uint8_t *>(c->v) + bytes, q ? c->k_exp + cells : nullptr, q ? c->v_exp + cells : nullptr,
                   c->n_kv, c->capacity, c->window, c->window ? c->sinks : 0u};
}

template <int HD>
cudaError_t launch_store(int elem, const StoreArgs &given, void *stream) {
    /* more query rows to a warp once there are warps enough: position, cos and sin are read once for them */
    StoreArgs a = given;
    a.chunks = (uint64_t)a.T * a.n_q * (HD / 8u) >= 1u << 20 ? 2u : 1u;
    const uint64_t units = (uint64_t)(store_groups<HD>(a.n_q, kStoreQ * a.chunks) + store_groups<HD>(a.c.n_kv, kStoreK) + store_groups<HD>(a.c.n_kv, kStoreV)) * a.T, blocks = (units + 7u) / 8u;
    if (units > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    const uint32_t threads = units >= 8u ? 256u : (uint32_t)units * 32u;
    const auto kernel = elem == kKvE4m3 ? (a.q_norm ? kv_store_kernel<HD, kKvE4m3, true> : kv_store_kernel<HD, kKvE4m3, false>)
                                        : (a.q_norm ? kv_store_kernel<HD, kKvBf16, true> : kv_store_kernel<HD, kKvBf16, false>);
    return launch(kernel, dim3((uint32_t)blocks), dim3(threads), stream, a);
}

}  // namespace

NWC_EXPORT int nwc_kv_append(void *stream, const nwc_kv_cache *cache, uint32_t layer, const uint16_t *qkv, uint64_t ldqkv, uint32_t T, uint32_t n_q,
                             const uint16_t *q_norm, const uint16_t *k_norm, const uint16_t *cos_t, const uint16_t *sin_t, uint32_t max_pos,
                             const int32_t *pos, const int32_t *depth, float eps, uint16_t *q_out, int *status) {
    if (!cache_ok(cache, layer, T) || !T || T > NWC_KV_MAX_TOKENS || !n_q || n_q % cache->n_kv || n_q > 65535u) return -1;
    if (!qkv || !cos_t || !sin_t || !pos || !q_out || !status || !q_norm != !k_norm) return -1;
    const uint64_t width = (uint64_t)(n_q + 2u * cache->n_kv) * cache->head_dim;
    if (ldqkv < width || ldqkv % 8u) return -1;
    if (!aligned16(qkv) || !aligned16(cos_t) || !aligned16(sin_t) || !aligned16(q_out) || !aligned16(q_norm) || !aligned16(k_norm)) return -1;
    const StoreArgs a{layer_of(cache, layer), qkv, ldqkv, T, n_q, q_norm, k_norm, cos_t, sin_t, max_pos, pos, depth, eps, q_out, status, 1u};
    return (int)(cache->head_dim == 64u ? launch_store<64>(cache->elem, a, stream) : cache->head_dim == 128u ? launch_store<128>(cache->elem, a, stream) : launch_store<256>(cache->elem, a, stream));
}

NWC_EXPORT int nwc_kv_read(void *stream, const nwc_kv_cache *cache, uint32_t layer, uint32_t first, uint32_t count, uint16_t *k_out, uint16_t *v_out) {
    if (!cache_ok(cache, layer, 0u) || !count || !k_out || !v_out || !aligned16(k_out) || !aligned16(v_out) || cache->n_kv > 65535u) return -1;
    const uint64_t end = (uint64_t)first + count;
    if (end > (cache->window ? 0x7FFFFFFFull : cache->capacity)) return -1;
    /* rows of the ring that one call asks for must be there at the same time */
    if (cache->window && end > cache->sinks && end - (first > cache->sinks ? first : cache->sinks) > cache->capacity - cache->sinks) return -1;
    const ReadArgs a{layer_of(cache, layer), first, count, cache->head_dim, k_out, v_out};
    const uint64_t threads = (uint64_t)count * (cache->head_dim >> 4);
    const dim3 grid((uint32_t)((threads + 255u) / 256u), cache->n_kv, 2u);
    return (int)(cache->elem == kKvE4m3 ? launch(kv_read_kernel<kKvE4m3>, grid, dim3(256), stream, a) : launch(kv_read_kernel<kKvBf16>, grid, dim3(256), stream, a));
}

NWC_EXPORT int nwc_kv_commit(void *stream, const nwc_kv_cache *cache, uint32_t T, const int32_t *pos, const int32_t *path, const int32_t *count, uint32_t most, int *status) {
    if (!cache_ok(cache, 0u, T) || !T || T > NWC_KV_MAX_TREE || most > T || !pos || !path || !count || !status) return -1;
    if (!most) return 0;
    const uint32_t row_bytes = cache->head_dim * (cache->elem == kKvBf16 ? 2u : 1u);
    return (int)launch(kv_commit_kernel, dim3(cache->layers * cache->n_kv), dim3(256), stream, layer_of(cache, 0u), row_bytes, T, pos, path, count, most, status);
}

NWC_EXPORT int nwc_kv_wait_probe(void *stream, int *status) { return status ? (int)launch_kv_wait_probe((cudaStream_t)stream, status) : -1; }

static uint64_t workspace_bytes(const KvPlan &p, uint32_t head_dim) { return p.cells * (head_dim + 2u) * sizeof(float); }

NWC_EXPORT uint64_t nwc_kv_attention_workspace(const nwc_kv_cache *cache, uint32_t T, uint32_t n_q) {
    if (!cache || !T || T > NWC_KV_MAX_TOKENS || !n_q || n_q > 65535u || !cache->n_kv || n_q % cache->n_kv) return 0;
    const int sms = nwc_setup();
    if (sms <= 0) return 0;
    return workspace_bytes(kv_attention_plan(cache->elem, cache->head_dim, cache->n_kv, cache->capacity, cache->window, cache->sinks, T, n_q, sms), cache->head_dim);
}

NWC_EXPORT int nwc_kv_attention(void *stream, const nwc_kv_cache *cache, uint32_t layer, const uint16_t *q, uint64_t ldq, uint32_t T, uint32_t n_q,
                                const int32_t *pos, const uint32_t *visible, const int32_t *depth, float scale, uint16_t *out, void *workspace,
                                uint64_t workspace_size, int *status) {
    if (!cache_ok(cache, layer, T) || !T || T > NWC_KV_MAX_TOKENS || !n_q || n_q % cache->n_kv || n_q > 65535u) return -1;
    if (!q || !pos || !out || !status || !aligned16(q) || !aligned16(out) || !aligned16(workspace) || ldq < (uint64_t)n_q * cache->head_dim || ldq % 8u) return -1;
    if (visible ? T > NWC_KV_MAX_TREE || !depth : depth != nullptr) return -1;
    if (!(scale > 0.f) || scale > 2e38f) return -1;                  /* (times log2(e) it is a number too) */
    const int sms = nwc_setup();
    if (sms <= 0) return (int)cudaErrorNoDevice;
    const KvPlan plan = kv_attention_plan(cache->elem, cache->head_dim, cache->n_kv, cache->capacity, cache->window, cache->sinks, T, n_q, sms);
    const uint64_t need = workspace_bytes(plan, cache->head_dim);
    if (need && (!workspace || workspace_size < need)) return -1;
    float *part_o = static_cast<float *>(workspace), *part_ml = need ? part_o + plan.cells * cache->head_dim : nullptr;
    const KvAttention a{layer_of(cache, layer), q, ldq, T, n_q, pos, visible, depth, scale * 1.4426950408889634f, out, status, part_o, part_ml, plan.splits, layer, cache->layers, 0u};
    return (int)launch_kv_attention((cudaStream_t)stream, cache->elem, cache->head_dim, a, plan, sms);
}
