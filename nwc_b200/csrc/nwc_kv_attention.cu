/* Attention of a few query rows over a cache of nwc_kv.h: o_t = sum over the positions p that token t sees of
 * softmax_p(scale q_t . k_p) v_p, grouped heads; zeros where a token sees nothing.
 *
 * What token t (position own = pos + t, or pos + depth[t] with a draft tree) sees:
 *   p < pos + T with p <= own (no tree) or p < pos or bit p - pos of visible[t] (tree); and, with a window and for p that are
 *   not drafted, p < sinks or p > own - window.
 *
 * One token reads every visible row once and computes little: the bound is the memory's rate.  So the rows of a key/value
 * head are read once for all of its query rows (T * group of them, 16 or 32 at a time: the M of mma.m16n8k16), the keys are
 * divided over the CTAs of the whole GPU, and every warp streams its own tiles through a ring of asynchronous copies in shared memory,
 * deep enough to keep the memory busy.  There is no barrier between the warps of a CTA until their shares are joined.
 *
 * Fragments.  A dot product may add its terms in any order, so the B fragment of K takes the 16-byte piece that a lane reads
 * from a key's row as it lies, and Q is laid out once to match; likewise the columns of V: the n-th column of an MMA is the
 * dimension that lane group n's piece holds at that place.  Neither K nor V is ever transposed or re-stored.
 *
 * bf16 caches take bf16 products.  e4m3 codes become f16 (exactly, one conversion for two codes; bf16 would take bit moves and a
 * multiplication, 640 instead of 230 of a tile's instructions, which now are 735 for 32 keys), with a query row scaled by a power of two to fill f16's range; the unit 2^e of a K row multiplies its scores, that of a V
 * row, relative to the largest that was met and seen so far, its weights.
 *
 * The weights are rounded for the second product: to bf16 (by up to 2^-8 of each), or, times the V rows' units, to f16.  A
 * weight is at most 2^8 and is scaled up by 2^7, so that f16 holds it to 2^-11 of itself down to 2^-21 (the running maximum's is 1), and to 2^-32
 * below.  Those absolute errors of a warp's N keys stay below 2^-12 of the row's sum of weights times units (N 2^-28 of it for N up
 * to 2^16) as long as that is 2^-4 and N 2^-20 or more; until it is (a sink with a value of zero, an outlier among the units),
 * tiles take bf16 products.  What f16 costs then is small beside the row as a whole, and not beside a dimension in which every
 * value of weight is a zero.
 * The sum of the weights, the running maximum and all accumulators are fp32.
 *
 * One token over 131071 e4m3 positions (64 + 8 heads of 128): 51.4 us, 5.3 TB/s, 0.82 of measured bandwidth.  What is left is
 * latency: three warps per scheduler (168 registers, rings that fill the shared memory) issue 2.0 instructions of 4 per clock,
 * and no pipe is above 46 %.
 */
#include "nwc_kv.h"
#include "nwc_async.cuh"
#include "nwc_launch.h"

namespace nwc {

namespace {

__device__ __forceinline__ void kv_dependency_sync() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { uint32_t d; asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a)); return d; }
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void mma16816_half(float (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t pack_half(float a, float b) { uint32_t d; asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a)); return d; }
/* four codes -> two f16 pairs (codes 0, 1 and 2, 3): exact */
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
/* codes (in the high bytes of both halves of w; the low bytes may hold anything) -> bf16 pair */
__device__ __forceinline__ uint32_t codes_to_bf16(uint32_t w) { return kv_mul2(((w >> 4) & 0x07F007F0u) | (w & 0x80008000u), kTwoTo120); }
constexpr int32_t kWeightBits = 7;                                   /* weights in f16 are held times 2^7 (they reach 2^8: 2^15 of f16's 2^16) */
/* 2^e for -126 <= e <= 127 */
__device__ __forceinline__ float power_of_two(int32_t e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__host__ __device__ constexpr uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

/* Shape of the few-rows kernel: warps that take tiles of kKeys keys, kStages of them in flight per warp.
   Long caches (SHORT = 0): one CTA per SM whose rings fill its shared memory; the CTAs' shares meet in a second kernel.
   Short ones (SHORT = 1): small tiles, so that the dependent chain of one warp is short, four warps, and the CTAs that divide
   one head's keys form a cluster that joins its shares through distributed shared memory: no second launch. */
template <int HD, int ELEM, int MT, int SHORT> struct Few {
    static constexpr uint32_t kRowBytes = HD * (ELEM == kKvE4m3 ? 1u : 2u);
    static constexpr uint32_t kKeys = ELEM == kKvE4m3 && !SHORT ? 32u : 16u;
    static constexpr uint32_t kStageBytes = 2u * kKeys * kRowBytes;                     /* K and V */
    static constexpr uint32_t kWarps = SHORT ? 4u : HD == 256 ? 6u : MT == 2 ? 8u : 12u, kStages = SHORT ? (ELEM == kKvE4m3 ? 4u : 3u) : HD == 64 ? 4u : MT == 2 ? 3u : 2u;
    static constexpr uint32_t kRows = 16u * MT;
    /* a row of a warp's outputs: ten floats for the eight columns of an accumulator, eight (mod 32) between rows: both the
       stores in fragment order and the loads in order of dimensions meet different banks */
    static constexpr uint32_t kPitch = (HD / 8u * 10u + 23u) / 32u * 32u + 8u;
    static constexpr uint32_t kRing = larger(kWarps * kStages * kStageBytes, kWarps * kRows * kPitch * 4u);
    static constexpr uint32_t kQ = kRing, kPart = kQ + kRows * HD * 2u, kQUnit = kPart + 2u * kWarps * kRows * 4u, kShare = (kQUnit + kRows * 4u + 15u) / 16u * 16u;
    static constexpr uint32_t kSmem = kShare + (SHORT ? kRows * (HD + 2u) * 4u + 16u * kRows * 8u : kRows * 8u);
};
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
    uint32_t there; float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

}  // namespace

template <int HD, int ELEM, int MT, int SHORT>
__global__ void __launch_bounds__(32 * Few<HD, ELEM, MT, SHORT>::kWarps, 1) kv_attention_few_kernel(const KvAttention a) {
    using F = Few<HD, ELEM, MT, SHORT>;
    constexpr uint32_t kRows = F::kRows, kNT = F::kKeys / 8u, kWarps = F::kWarps;
    extern __shared__ __align__(128) uint8_t few_raw[];
    const uint32_t ring = smem_addr(few_raw), tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, g = lane >> 2, c = lane & 3u;
    uint8_t *qs = few_raw + F::kQ;                                                  /* Q in fragment order: [kSteps][MT][32 lanes] uint4 */
    const uint32_t mine = ring + warp * F::kStages * F::kStageBytes;
    float *part_m = reinterpret_cast<float *>(few_raw + F::kPart), *part_l = part_m + kWarps * kRows, *q_unit = reinterpret_cast<float *>(few_raw + F::kQUnit);
    const uint32_t group = a.n_q / a.c.n_kv, rows = a.T * group, kvh = blockIdx.x % a.c.n_kv, row0 = (blockIdx.x / a.c.n_kv) * kRows, split = blockIdx.y;
    kv_dependency_sync();
    const int32_t pos = *a.pos;
    if (pos < 0 || (uint64_t)pos + a.T > (a.c.window ? 0x7FFFFFFFu : a.c.capacity)) { if (tid == 0) atomicOr(a.status, kKvStatusPosition); return; }
    const KvSpan span = kv_span(pos, a.T, a.c.window, a.c.sinks);
    /* this CTA's keys, in tiles of kKeys; tile i of a warp is the CTA's tile warp + i * kWarps */
    const uint32_t all_tiles = (span.count + F::kKeys - 1u) / F::kKeys, first_tile = (uint32_t)((uint64_t)all_tiles * split / a.splits), last_tile = (uint32_t)((uint64_t)all_tiles * (split + 1u) / a.splits);
    const uint32_t my_tiles = last_tile - first_tile > warp ? (last_tile - first_tile - warp + kWarps - 1u) / kWarps : 0u;
    auto position = [&](uint32_t i) { return i < span.lead ? i : span.first + (i - span.lead); };
    auto slot_of = [&](uint32_t i) { return kv_slot(position(i), a.c.capacity, a.c.window, a.c.sinks); };
    /* The copies are 16 bytes per lane.  Pieces of a row change places so that the lanes of a quarter warp, which read K at four
       pieces of two rows and V at two pieces of four, meet eight different bank groups: piece ^ 4 in odd rows of K, piece ^ (row &
       6) in V.  (Bulk copies lay the rows down as they are: 63 us for 131071 e4m3 positions where this takes 53.) */
    constexpr uint32_t kCopies = F::kKeys * F::kRowBytes / 512u;      /* per lane and plane */
    auto k_place = [](uint32_t row, uint32_t piece) { return row * F::kRowBytes + ((F::kRowBytes >= 128u ? piece ^ ((row & 1u) << 2) : piece) << 4); };
    auto v_place = [](uint32_t row, uint32_t piece) {
        if (F::kRowBytes >= 128u) return row * F::kRowBytes + ((piece ^ (row & 6u)) << 4);
        return (row >> 1) * 128u + (((((row & 1u) << 2) | piece) ^ (row & 6u)) << 4);          /* 64-byte rows: two of them share a line */
    };
    auto issue = [&](uint32_t i) {
        const uint32_t s = i % F::kStages, key0 = (first_tile + warp + i * kWarps) * F::kKeys, n = min(F::kKeys, span.count - key0);
        const uint32_t dst = mine + s * F::kStageBytes;
        const uint64_t cell = (uint64_t)kvh * a.c.capacity;
        const uint32_t a0 = slot_of(key0);
        if (n == F::kKeys && slot_of(key0 + n - 1u) == a0 + n - 1u) {                   /* neither the end of the sinks nor of the ring inside */
            const uint8_t *kf = a.c.k + (cell + a0) * F::kRowBytes + lane * 16u, *vf = a.c.v + (cell + a0) * F::kRowBytes + lane * 16u;
#pragma unroll
            for (uint32_t e = 0; e < kCopies; e++) {
                const uint32_t at = e * 512u + lane * 16u, row = at / F::kRowBytes, piece = (at % F::kRowBytes) >> 4;
                copy16(dst + k_place(row, piece), kf + e * 512u, 16u);
                copy16(dst + F::kKeys * F::kRowBytes + v_place(row, piece), vf + e * 512u, 16u);
            }
        } else {
#pragma unroll
            for (uint32_t e = 0; e < kCopies; e++) {                                    /* rows behind the last key arrive as zeros: weight 0 times whatever lies there must be 0 */
                const uint32_t at = e * 512u + lane * 16u, row = at / F::kRowBytes, piece = (at % F::kRowBytes) >> 4;
                const uint64_t from = (cell + (row < n ? slot_of(key0 + row) : 0u)) * F::kRowBytes + piece * 16u;
                copy16(dst + k_place(row, piece), a.c.k + from, row < n ? 16u : 0u);
                copy16(dst + F::kKeys * F::kRowBytes + v_place(row, piece), a.c.v + from, row < n ? 16u : 0u);
            }
        }
    };
    /* the exponent bytes of the key that this lane stands for in tile i (a tile early; behind the last key, the last one's) */
    uint8_t k_next = 0, v_next = 0;
    auto units = [&](uint32_t i) {
        if (ELEM != kKvE4m3) return;
        const uint64_t cell = (uint64_t)kvh * a.c.capacity + slot_of(min((first_tile + warp + i * kWarps) * F::kKeys + lane, span.count - 1u));
        k_next = a.c.k_exp[cell]; v_next = a.c.v_exp[cell];
    };
    for (uint32_t i = 0; i < F::kStages; i++) { if (i < my_tiles) issue(i); copies_commit(); }
    units(0u);
    /* Q: the 16-byte piece of a row that meets the K piece of lane c, in the order its words are used.  A row is one warp's. */
    for (uint32_t r = warp; r < kRows; r += kWarps) {
        const uint32_t row = row0 + r;
        uint32_t w[HD / 64];
        float top = 0.f;
#pragma unroll
        for (uint32_t j = 0; j < HD / 64u; j++) {                                       /* dimensions 2 (32 j + lane), + 1 */
            w[j] = row < rows ? *reinterpret_cast<const uint32_t *>(a.q + (uint64_t)(row / group) * a.ldq + (uint64_t)(kvh * group + row % group) * HD + 64u * j + 2u * lane) : 0u;
            top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[j] << 16)), fabsf(__uint_as_float(w[j] & 0xFFFF0000u))));
        }
        if (ELEM == kKvE4m3) {
            /* largest magnitude into [2^14, 2^15): a number 2^-29 of it is still held to bf16's precision */
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const int32_t e = max((int32_t)(__float_as_uint(top) >> 23) - 127, -100);
            const float up = power_of_two(14 - e);
            if (lane == 0) q_unit[r] = power_of_two(e - 14);
#pragma unroll
            for (uint32_t j = 0; j < HD / 64u; j++) w[j] = pack_half(__uint_as_float(w[j] << 16) * up, __uint_as_float(w[j] & 0xFFFF0000u) * up);
        }
#pragma unroll
        for (uint32_t j = 0; j < HD / 64u; j++) {
            const uint32_t d = 64u * j + 2u * lane;
            uint32_t step, cc;
            if (ELEM == kKvE4m3) { step = (d >> 6) * 4u + ((d & 15u) >> 2); cc = (d >> 4) & 3u; } else { step = (d >> 5) * 2u + ((d & 7u) >> 2); cc = (d >> 3) & 3u; }
            /* a0 a1 a2 a3 = (row g, first pair) (row g + 8, first) (g, second) (g + 8, second) */
            reinterpret_cast<uint32_t *>(qs)[((step * MT + (r >> 4)) * 32u + (r & 7u) * 4u + cc) * 4u + ((d >> 1) & 1u) * 2u + ((r >> 3) & 1u)] = w[j];
        }
    }
    __syncthreads();
    /* this lane's rows: token and own position */
    float row_scale[2 * MT];
    uint32_t token[2 * MT], own[2 * MT], top_byte = 0u, own_min = 0xFFFFFFFFu, own_max = 0u;
#pragma unroll
    for (uint32_t i = 0; i < 2u * MT; i++) {
        const uint32_t row = min(row0 + (i >> 1) * 16u + (i & 1u) * 8u + g, rows - 1u);
        token[i] = row / group;
        own[i] = (uint32_t)pos + (a.depth ? (uint32_t)a.depth[token[i]] : token[i]);
        own_min = min(own_min, own[i]); own_max = max(own_max, own[i]);
        row_scale[i] = ELEM == kKvE4m3 ? a.scale * q_unit[(i >> 1) * 16u + (i & 1u) * 8u + g] : a.scale;
    }
    own_max = __reduce_max_sync(0xffffffffu, own_max); own_min = __reduce_min_sync(0xffffffffu, own_min);
    const uint32_t open_end = a.visible ? (uint32_t)pos : own_min + 1u;                 /* positions below it are seen by every row, window apart */
    const uint32_t words = (a.T + 31u) / 32u;
    float o[MT][HD / 8][4], m[2 * MT], l[2 * MT], held[2 * MT];                         /* held (e4m3): weights times units, as scaled for f16, of this lane's keys */
    bool settled = false;                                                               /* every row holds at least `enough` */
    const float enough = fmaxf(0x1p-4f, (float)my_tiles * (float)F::kKeys * 0x1p-20f) * (float)(1 << kWeightBits);
#pragma unroll
    for (uint32_t i = 0; i < MT; i++)
#pragma unroll
        for (uint32_t j = 0; j < HD / 8u; j++)
#pragma unroll
            for (uint32_t e = 0; e < 4u; e++) o[i][j][e] = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < 2u * MT; i++) { m[i] = -INFINITY; l[i] = held[i] = 0.f; }
    for (uint32_t it = 0; it < my_tiles; it++) {
        const uint32_t s = it % F::kStages, key0 = (first_tile + warp + it * kWarps) * F::kKeys, n = min(F::kKeys, span.count - key0);
        const uint32_t kt = mine + s * F::kStageBytes, vt = kt + F::kKeys * F::kRowBytes;
        const uint32_t k_byte = k_next, v_byte = v_next;
        copies_wait<F::kStages - 1u>();                                                 /* this lane's copies of the tile ... */
        __syncwarp();                                                                   /* ... and the other lanes' */
        units(it + 1u);
        /* scores */
        float sc[MT][kNT][4];
#pragma unroll
        for (uint32_t i = 0; i < MT; i++)
#pragma unroll
            for (uint32_t j = 0; j < kNT; j++)
#pragma unroll
                for (uint32_t e = 0; e < 4u; e++) sc[i][j][e] = 0.f;
        constexpr uint32_t kPieces = F::kRowBytes / 64u, kStepsPerPiece = ELEM == kKvE4m3 ? 4u : 2u;
#pragma unroll
        for (uint32_t pc = 0; pc < kPieces; pc++) {
            uint4 qf[kStepsPerPiece][MT];
#pragma unroll
            for (uint32_t st = 0; st < kStepsPerPiece; st++)
#pragma unroll
                for (uint32_t i = 0; i < MT; i++) qf[st][i] = reinterpret_cast<const uint4 *>(qs)[((pc * kStepsPerPiece + st) * MT + i) * 32u + lane];
#pragma unroll
            for (uint32_t j = 0; j < kNT; j++) {
                const uint4 w = lds128(kt + j * 8u * F::kRowBytes + k_place(g, pc * 4u + c));
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
                if (ELEM == kKvE4m3) {
#pragma unroll
                    for (uint32_t st = 0; st < kStepsPerPiece; st++) {
                        uint32_t b0, b1;
                        codes_to_half(u[st], b0, b1);
#pragma unroll
                        for (uint32_t i = 0; i < MT; i++) mma16816_half(sc[i][j], qf[st][i], b0, b1);
                    }
                } else {
#pragma unroll
                    for (uint32_t st = 0; st < 2u; st++)
#pragma unroll
                        for (uint32_t i = 0; i < MT; i++) mma16816(sc[i][j], qf[st][i], u[2 * st], u[2 * st + 1]);
                }
            }
        }
        /* log2 scores, masked; a tile that every row sees whole needs no mask */
        const uint32_t p_first = position(key0), p_last = position(key0 + n - 1u);
        const bool open = n == F::kKeys && p_last < open_end && (!a.c.window || p_last < a.c.sinks || (p_first > own_max || own_max - p_first < a.c.window));
        const float k_unit = kv_unit(k_byte);
#pragma unroll
        for (uint32_t j = 0; j < kNT; j++)
#pragma unroll
            for (uint32_t b = 0; b < 2u; b++) {
                const float f = ELEM == kKvE4m3 ? __shfl_sync(0xffffffffu, k_unit, j * 8u + 2u * c + b) : 1.f;
#pragma unroll
                for (uint32_t i = 0; i < 2u * MT; i++) {
                    float &x = sc[i >> 1][j][2u * (i & 1u) + b];
                    x *= ELEM == kKvE4m3 ? f * row_scale[i] : row_scale[i];
                }
            }
        uint32_t seen = F::kKeys == 32u ? 0xFFFFFFFFu : 0xFFFFu;                        /* (e4m3) keys of the tile that some row sees */
        if (!open) {
            seen = 0u;
#pragma unroll
            for (uint32_t j = 0; j < kNT; j++)
#pragma unroll
                for (uint32_t b = 0; b < 2u; b++) {
                    const uint32_t kk = j * 8u + 2u * c + b, p = position(key0 + kk);
#pragma unroll
                    for (uint32_t i = 0; i < 2u * MT; i++) {
                        bool sees = kk < n && (!a.c.window || p < a.c.sinks || p + a.c.window > own[i]);
                        if (!a.visible) sees = sees && p <= own[i];
                        else if (p >= (uint32_t)pos && kk < n) { const uint32_t d = p - (uint32_t)pos; sees = (a.visible[(uint64_t)token[i] * words + (d >> 5)] >> (d & 31u)) & 1u; }
                        if (!sees) sc[i >> 1][j][b + 2u * (i & 1u)] = -INFINITY;
                        else seen |= 1u << kk;
                    }
                }
            if (ELEM == kKvE4m3) seen = __reduce_or_sync(0xffffffffu, seen);
        }
        /* running maximum: raised (and the sums rescaled) only when some row's tile maximum passes it by more than 2^8, so
           weights stay below 2^8 and the rescaling is rare */
        bool raise = false;
        float top[2 * MT];
#pragma unroll
        for (uint32_t i = 0; i < 2u * MT; i++) {
            float t = -INFINITY;
#pragma unroll
            for (uint32_t j = 0; j < kNT; j++) t = fmaxf(t, fmaxf(sc[i >> 1][j][2u * (i & 1u)], sc[i >> 1][j][2u * (i & 1u) + 1u]));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1)); t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
            top[i] = t; raise = raise || t > m[i] + 8.f;
        }
        /* the same for the largest unit of the V rows that are seen: weights are multiplied by 2^(v_seen - top_byte) <= 1 */
        const uint32_t v_seen = (seen >> lane) & 1u ? v_byte : 0u;
        uint32_t byte_up = top_byte;
        if (ELEM == kKvE4m3) { byte_up = max(top_byte, __reduce_max_sync(0xffffffffu, v_seen)); raise = raise || byte_up != top_byte; }
        if (__any_sync(0xffffffffu, raise)) {
            const float v_down = ELEM == kKvE4m3 ? power_of_two(max((int32_t)(top_byte - byte_up), -126)) : 1.f;
            top_byte = byte_up; settled = false;
#pragma unroll
            for (uint32_t i = 0; i < 2u * MT; i++) {
                const float up = fmaxf(m[i], top[i]), f = up == -INFINITY ? 1.f : exp2_fast(m[i] - up);
                m[i] = up; l[i] *= f;
                const float fo = f * v_down;
                held[i] *= fo;
#pragma unroll
                for (uint32_t j = 0; j < HD / 8u; j++) { o[i >> 1][j][2u * (i & 1u)] *= fo; o[i >> 1][j][2u * (i & 1u) + 1u] *= fo; }
            }
        }
        float base[2 * MT];
#pragma unroll
        for (uint32_t i = 0; i < 2u * MT; i++) base[i] = m[i] == -INFINITY ? 0.f : m[i];
        const float v_unit = power_of_two(max((int32_t)(v_seen - top_byte), -126) + kWeightBits);
#pragma unroll
        for (uint32_t j = 0; j < kNT; j++)
#pragma unroll
            for (uint32_t b = 0; b < 2u; b++) {
                const float vu = ELEM == kKvE4m3 ? __shfl_sync(0xffffffffu, v_unit, j * 8u + 2u * c + b) : 1.f;
#pragma unroll
                for (uint32_t i = 0; i < 2u * MT; i++) {
                    float &x = sc[i >> 1][j][2u * (i & 1u) + b];
                    x = exp2_fast(x - base[i]);
                    l[i] += x;
                    if (ELEM == kKvE4m3) x *= vu;
                }
            }
        /* bf16 products for a tile while some row holds too little for f16 (a row that holds nothing has no weights yet) */
        bool wide = false;
        if (ELEM == kKvE4m3 && !settled) {
            bool all = true;
#pragma unroll
            for (uint32_t i = 0; i < 2u * MT; i++) {
#pragma unroll
                for (uint32_t j = 0; j < kNT; j++) held[i] += sc[i >> 1][j][2u * (i & 1u)] + sc[i >> 1][j][2u * (i & 1u) + 1u];
                float sum = held[i] + __shfl_xor_sync(0xffffffffu, held[i], 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                all = all && sum >= enough; wide = wide || (sum != 0.f && !(sum >= enough));
            }
            settled = __all_sync(0xffffffffu, all); wide = __any_sync(0xffffffffu, wide);
        }
        /* o += P V, 16 keys at a time; lane (g, c) holds keys 2c, 2c + 1, 2c + 8, 2c + 9 of the columns of piece g */
#pragma unroll
        for (uint32_t h = 0; h < kNT / 2u; h++) {
            uint4 pf[MT];
#pragma unroll
            for (uint32_t i = 0; i < MT; i++) {
                auto pack = [&](float x, float y) { return ELEM == kKvE4m3 && !wide ? pack_half(x, y) : pack_bf16(x, y); };
                pf[i] = make_uint4(pack(sc[i][2 * h][0], sc[i][2 * h][1]), pack(sc[i][2 * h][2], sc[i][2 * h][3]),
                                   pack(sc[i][2 * h + 1][0], sc[i][2 * h + 1][1]), pack(sc[i][2 * h + 1][2], sc[i][2 * h + 1][3]));
            }
            const uint32_t v0 = vt + h * 16u * F::kRowBytes;
            constexpr uint32_t kPieceDims = ELEM == kKvE4m3 ? (HD == 64 ? 8u : 16u) : 8u, kVPieces = HD / (8u * kPieceDims);
#pragma unroll
            for (uint32_t pc = 0; pc < kVPieces; pc++) {
                uint32_t w[4][4];                                                       /* [key][word] */
#pragma unroll
                for (uint32_t e = 0; e < 4u; e++) {
                    const uint32_t row = 2u * c + (e & 1u), below = (e >> 1) * 8u * F::kRowBytes;       /* (eight rows on, the places are the same) */
                    if (ELEM == kKvE4m3 && HD == 64) { const uint2 x = lds64(v0 + below + v_place(row, g >> 1) + (g & 1u) * 8u); w[e][0] = x.x; w[e][1] = x.y; }
                    else { const uint4 x = lds128(v0 + below + v_place(row, pc * 8u + g)); w[e][0] = x.x; w[e][1] = x.y; w[e][2] = x.z; w[e][3] = x.w; }
                }
                if (ELEM == kKvE4m3 && wide) {
#pragma unroll
                    for (uint32_t d = 0; d < kPieceDims; d++) {
                        const uint32_t sel = (d & 3u) << 4 | ((d & 3u) + 4u) << 12;
                        const uint32_t b0 = codes_to_bf16(__byte_perm(w[0][d >> 2], w[1][d >> 2], sel)), b1 = codes_to_bf16(__byte_perm(w[2][d >> 2], w[3][d >> 2], sel));
#pragma unroll
                        for (uint32_t i = 0; i < MT; i++) mma16816(o[i][pc * kPieceDims + d], pf[i], b0, b1);
                    }
                } else if (ELEM == kKvE4m3) {
#pragma unroll
                    for (uint32_t d = 0; d < kPieceDims; d += 2u) {
                        /* bytes d % 4 and d % 4 + 1 of the two keys' words, side by side */
                        const uint32_t sel = d & 2u ? 0x7362u : 0x5140u;
                        uint32_t b0[2], b1[2];
                        codes_to_half(__byte_perm(w[0][d >> 2], w[1][d >> 2], sel), b0[0], b0[1]);
                        codes_to_half(__byte_perm(w[2][d >> 2], w[3][d >> 2], sel), b1[0], b1[1]);
#pragma unroll
                        for (uint32_t x = 0; x < 2u; x++)
#pragma unroll
                            for (uint32_t i = 0; i < MT; i++) mma16816_half(o[i][pc * kPieceDims + d + x], pf[i], b0[x], b1[x]);
                    }
                } else {
#pragma unroll
                    for (uint32_t d = 0; d < 8u; d++) {
                        const uint32_t sel = d & 1u ? 0x7632u : 0x5410u;
                        const uint32_t b0 = __byte_perm(w[0][d >> 1], w[1][d >> 1], sel), b1 = __byte_perm(w[2][d >> 1], w[3][d >> 1], sel);
#pragma unroll
                        for (uint32_t i = 0; i < MT; i++) mma16816(o[i][pc * 8u + d], pf[i], b0, b1);
                    }
                }
            }
        }
        __syncwarp();
        if (it + F::kStages < my_tiles) issue(it + F::kStages);
        copies_commit();
    }
    /* join the warps: common maximum, then sums and outputs rescaled to it, in warp order */
#pragma unroll
    for (uint32_t i = 0; i < 2u * MT; i++) { l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1); l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2); }
    const uint32_t live = min(kRows, rows - row0);                                      /* rows of this tile that exist */
    __syncthreads();                                                                    /* every warp has done with its ring: O goes there */
    float *part = reinterpret_cast<float *>(few_raw);                                   /* [kWarps][kRows][kPitch] */
    constexpr uint32_t kPieceDims = ELEM == kKvE4m3 ? (HD == 64 ? 8u : 16u) : 8u;
    const float o_unit = ELEM == kKvE4m3 ? kv_unit(top_byte) * (1.f / (1 << kWeightBits)) : 1.f;
#pragma unroll
    for (uint32_t i = 0; i < 2u * MT; i++) {
        const uint32_t r = (i >> 1) * 16u + (i & 1u) * 8u + g;
        if (c == 0) { part_m[warp * kRows + r] = m[i]; part_l[warp * kRows + r] = l[i]; }
        if (r < live && m[i] != -INFINITY) {
            float *to = part + (warp * kRows + r) * F::kPitch + 2u * c;
#pragma unroll
            for (uint32_t j = 0; j < HD / 8u; j++) *reinterpret_cast<float2 *>(to + j * 10u) = make_float2(o[i >> 1][j][2u * (i & 1u)] * o_unit, o[i >> 1][j][2u * (i & 1u) + 1u] * o_unit);
        }
    }
    __syncthreads();
    float *share = reinterpret_cast<float *>(few_raw + F::kShare), *share_ml = share + (SHORT ? kRows * HD : 0u);      /* [kRows][HD] (a cluster's only), [kRows][2] */
    if (tid < kRows) {
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; w++) top = fmaxf(top, part_m[w * kRows + tid]);
#pragma unroll
        for (uint32_t w = 0; w < kWarps; w++) {
            const float mw = part_m[w * kRows + tid], f = mw == -INFINITY ? 0.f : exp2_fast(mw - top);
            total = fmaf(part_l[w * kRows + tid], f, total);
            part_m[w * kRows + tid] = f;                                                /* from here on the warp's factor */
        }
        share_ml[2u * tid] = total == total ? top : 0.f; share_ml[2u * tid + 1u] = total;      /* (a query that is not a number has no maximum, but its share counts) */
    }
    __syncthreads();
    for (uint32_t at = tid; at < live * HD; at += 32u * kWarps) {
        const uint32_t r = at / HD, d = at % HD, row = row0 + r;
        /* dimension d = place d % kPieceDims of piece (d / kPieceDims) % 8: accumulator j, column d / kPieceDims % 8 */
        const uint32_t j = d / (8u * kPieceDims) * kPieceDims + d % kPieceDims, x = j * 10u + (d / kPieceDims) % 8u;
        float sum = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; w++) {
            const float f = part_m[w * kRows + r];
            if (f != 0.f) sum = fmaf(part[(w * kRows + r) * F::kPitch + x], f, sum);
        }
        const uint64_t line = (uint64_t)(row / group) * a.n_q + kvh * group + row % group;
        if (a.splits == 1u) {
            const float total = share_ml[2u * r + 1u];
            a.out[line * HD + d] = __bfloat16_as_ushort(__float2bfloat16_rn(total == 0.f ? 0.f : sum / total));
        } else if (SHORT) share[at] = sum;
        else {
            const uint64_t cell = (uint64_t)split * a.T * a.n_q + line;
            a.part_o[cell * HD + d] = sum;
            if (d == 0) *reinterpret_cast<float2 *>(a.part_ml + cell * 2u) = make_float2(share_ml[2u * r], share_ml[2u * r + 1u]);
        }
    }
    if (SHORT && a.splits > 1u) {
        /* join the CTAs of the cluster: each takes its part of the outputs, reading the others' shares; rank order */
        cluster_barrier();
        float2 *ml = reinterpret_cast<float2 *>(share_ml + 2u * kRows);                /* [16][kRows] */
        const uint32_t from = smem_addr(share), from_ml = smem_addr(share_ml);
        for (uint32_t e = tid; e < a.splits * live; e += 32u * kWarps) {
            const uint32_t y = e / live, r = e % live;
            ml[y * kRows + r] = make_float2(ld_cluster(from_ml + r * 8u, y), ld_cluster(from_ml + r * 8u + 4u, y));
        }
        __syncthreads();
        for (uint32_t at = split * 32u * kWarps + tid; at < live * HD; at += a.splits * 32u * kWarps) {
            const uint32_t r = at / HD, d = at % HD, row = row0 + r;
            float top = -INFINITY, total = 0.f, sum = 0.f;
            for (uint32_t y = 0; y < a.splits; y++) top = fmaxf(top, ml[y * kRows + r].x);
#pragma unroll 4
            for (uint32_t y = 0; y < a.splits; y++) {
                const float2 w = ml[y * kRows + r];
                const float f = w.x == -INFINITY ? 0.f : exp2_fast(w.x - top);
                total = fmaf(w.y, f, total); sum = fmaf(ld_cluster(from + at * 4u, y), f, sum);
            }
            const uint64_t line = (uint64_t)(row / group) * a.n_q + kvh * group + row % group;
            a.out[line * HD + d] = __bfloat16_as_ushort(__float2bfloat16_rn(total == 0.f ? 0.f : sum / total));
        }
        cluster_barrier();                                                              /* nobody leaves while its share is being read */
    }
}

/* The shares of the splits joined: `ways` warps per output row and 128 (64) of its dimensions take the splits in turn, and meet
   in shared memory in their order.  (One warp alone reads one share after another: 148 of them took 22 us.) */
template <int HD>
__global__ void __launch_bounds__(256) kv_attention_join_kernel(const KvAttention a, uint32_t ways) {
    constexpr uint32_t kPer = HD >= 128 ? 4u : 2u, kPieces = HD / (32u * kPer);
    __shared__ float sums[8][32u * kPer + 1u];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, way = warp % ways;
    const uint64_t unit = (uint64_t)blockIdx.x * (8u / ways) + warp / ways, lines = (uint64_t)a.T * a.n_q, line = unit / kPieces;
    const uint32_t d = (uint32_t)(unit % kPieces) * 32u * kPer + lane * kPer;
    kv_dependency_sync();
    const int32_t pos = *a.pos;
    if (pos < 0 || (uint64_t)pos + a.T > (a.c.window ? 0x7FFFFFFFu : a.c.capacity)) return;
    const bool live = line < lines;
    float top = -INFINITY, total = 0.f, sum[kPer];
#pragma unroll
    for (uint32_t j = 0; j < kPer; j++) sum[j] = 0.f;
    if (live) {
        for (uint32_t s = lane; s < a.splits; s += 32u) top = fmaxf(top, __ldcg(a.part_ml + ((uint64_t)s * lines + line) * 2u));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
#pragma unroll 4
        for (uint32_t s = way; s < a.splits; s += ways) {
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(a.part_ml) + (uint64_t)s * lines + line);
            const float *from = a.part_o + ((uint64_t)s * lines + line) * HD + d;
            float x[kPer];
            if (kPer == 4u) { const float4 v = __ldcg(reinterpret_cast<const float4 *>(from)); x[0] = v.x; x[1] = v.y; x[kPer - 2] = v.z; x[kPer - 1] = v.w; }
            else { const float2 v = __ldcg(reinterpret_cast<const float2 *>(from)); x[0] = v.x; x[1] = v.y; }
            if (ml.x == -INFINITY) continue;                                            /* (such a share has no outputs) */
            const float f = exp2_fast(ml.x - top);
            total = fmaf(ml.y, f, total);
#pragma unroll
            for (uint32_t j = 0; j < kPer; j++) sum[j] = fmaf(x[j], f, sum[j]);
        }
    }
    if (ways > 1u) {
#pragma unroll
        for (uint32_t j = 0; j < kPer; j++) sums[warp][lane * kPer + j] = sum[j];
        if (lane == 0) sums[warp][32u * kPer] = total;
        __syncthreads();
        if (way) return;
        for (uint32_t w = 1; w < ways; w++) {
            total += sums[warp + w][32u * kPer];
#pragma unroll
            for (uint32_t j = 0; j < kPer; j++) sum[j] += sums[warp + w][lane * kPer + j];
        }
    }
    if (!live) return;
    const float r = total == 0.f ? 0.f : 1.f / total;
    uint16_t *to = a.out + line * HD + d;
#pragma unroll
    for (uint32_t j = 0; j < kPer; j += 2u) *reinterpret_cast<uint32_t *>(to + j) = pack_bf16(sum[j] * r, sum[j + 1] * r);
}

namespace {

template <class... Params, class... Args>
cudaError_t launch(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool dependent, uint32_t cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    uint32_t n = 0;
    if (dependent) { attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[n++].val.programmaticStreamSerializationAllowed = 1; }
    if (cluster > 1u) { attr[n].id = cudaLaunchAttributeClusterDimension; attr[n].val.clusterDim.x = 1; attr[n].val.clusterDim.y = cluster; attr[n++].val.clusterDim.z = 1; }
    cfg.attrs = attr; cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

template <int HD, int ELEM, int MT, int SHORT>
cudaError_t launch_few(cudaStream_t st, const KvAttention &a) {
    using F = Few<HD, ELEM, MT, SHORT>;
    const uint32_t rows = a.T * (a.n_q / a.c.n_kv), tiles = (rows + F::kRows - 1u) / F::kRows;
    return launch(kv_attention_few_kernel<HD, ELEM, MT, SHORT>, dim3(a.c.n_kv * tiles, a.splits), dim3(32u * F::kWarps), F::kSmem, st, dependent_launch(), SHORT ? a.splits : 1u, a);
}
template <int HD, int ELEM>
cudaError_t launch_all(cudaStream_t st, const KvAttention &a, const KvPlan &p) {
    const uint32_t rows = a.T * (a.n_q / a.c.n_kv);
    const bool in_clusters = p.in_clusters;
    cudaError_t err;
    if (in_clusters) err = launch_few<HD, ELEM, 1, 1>(st, a);
    else if constexpr (HD != 256 && ELEM == kKvE4m3) err = rows > 16u /* the plan lets no more than 32 come here */ ? launch_few<HD, ELEM, 2, 0>(st, a) : launch_few<HD, ELEM, 1, 0>(st, a);
    else err = launch_few<HD, ELEM, 1, 0>(st, a);
    if (err != cudaSuccess || a.splits == 1u || in_clusters) return err;
    const uint64_t units = (uint64_t)a.T * a.n_q * (HD >= 128 ? HD / 128 : 1);
    const uint32_t ways = a.splits >= 16u ? 8u : a.splits >= 8u ? 4u : 1u, per_block = 8u / ways;
    /* (an ordinary dependent launch: the join's set-up overlaps the last CTAs; it waits for the whole grid before it reads) */
    return launch(kv_attention_join_kernel<HD>, dim3((uint32_t)((units + per_block - 1u) / per_block)), dim3(256), 0, st, true, 1u, a, ways);
}
template <int HD, int ELEM, int MT, int SHORT> void configure_one() {
    cudaFuncSetAttribute(kv_attention_few_kernel<HD, ELEM, MT, SHORT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Few<HD, ELEM, MT, SHORT>::kSmem);
    if (SHORT) cudaFuncSetAttribute(kv_attention_few_kernel<HD, ELEM, MT, SHORT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}
template <int HD> void configure_few() {
    configure_one<HD, kKvBf16, 1, 0>(); configure_one<HD, kKvBf16, 1, 1>(); configure_one<HD, kKvE4m3, 1, 0>(); configure_one<HD, kKvE4m3, 1, 1>();
    if constexpr (HD != 256) configure_one<HD, kKvE4m3, 2, 0>();
}

}  // namespace

/* Which kernel and how many CTAs.  Times in us on B200, eight key/value heads, calls of one kind in a graph:
     rows per key/value head   keys     head_dim 128:  e4m3 few / many   bf16 few / many     64:  e4m3 few / many   bf16 few / many
     16                        1024                    11.0 / 15.7       9.0 / 12.2               8.7 / 11.1        7.6 / 10.5
     16                        32768                   23 / 46           33 / 34                  17 / 30           16 / 25
     32                        1024                    18 / 14           18 / 14                  9.3 / 11.2        8.3 / 10.8
     32                        4096                    25 / 17           24 / 17                  12.3 / 13.6       10.7 / 12.8
     32                        32768                   31 / 44           42 / 35                  23 / 30           27 / 25
     32                        131072                  80 / 145          107 / 91                 59 / 111          68 / 61
     48                        32768                   45 / 44           59 / 36                  33 / 31           38 / 26
   The many-rows kernel multiplies 128 rows whatever there are, on tensor cores that make nothing of it, but it takes a while to
   fill and widens e4m3 rows at a rate of its own: the few-rows kernel takes up to 16 rows, and up to 32 of a long e4m3 cache.
   (Heads of 64 would gain 1 to 3 us over short caches with a border of 32.)
   head_dim 256 has no many-rows kernel: scores and outputs of two streams pass the tensor memory.  Its chunks and trees go
   through the few-rows kernel, 16 rows and the keys of the whole call per CTA: 2048 tokens of 8 + 2 heads over 8192 positions
   take 802 us (bf16; 77 with head_dim 128), 4096 tokens under a window of 64 1026 us. */
KvPlan kv_attention_plan(int elem, uint32_t head_dim, uint32_t n_kv, uint32_t capacity, uint32_t window, uint32_t sinks, uint32_t T, uint32_t n_q, int sms) {
    const uint32_t rows = T * (n_q / n_kv);
    const uint64_t keys = window ? (uint64_t)sinks + window + T - 1u : capacity;
    const bool longer = keys > kKvShortKeys;
    KvPlan p{1u, false, head_dim != 256u && rows > (elem == kKvE4m3 && longer ? 32u : 16u), 0u};
    if (p.many) {
        /* a CTA per SM, each with at least two tiles of 128 keys */
        const uint64_t ctas = (uint64_t)n_kv * ((rows + 255u) / 256u), seen = window ? (uint64_t)sinks + window + (T < 256u ? T : 256u) : capacity;
        const uint64_t most = (seen + 255u) / 256u, want = ctas < (uint64_t)sms ? (uint64_t)sms / ctas : 1u;
        p.splits = (uint32_t)(want < most ? want : most);
        p.cells = p.splits > 1u ? (uint64_t)p.splits * ctas * 256u : 0u;
        return p;
    }
    const uint32_t per = head_dim == 256u || rows <= 16u ? 16u : 32u;
    const uint64_t ctas = (uint64_t)n_kv * ((rows + per - 1u) / per);
    if (ctas >= (uint64_t)sms * 2u) return p;
    if (!longer) {
        /* Clusters of 2^k CTAs, a tile of 16 keys for each of their four warps, as long as the GPU has room for them side by
           side: up to 5/4 CTAs per SM (bf16, 4096 keys, up to 1, 5/4 and 2: ten key/value heads 9.9, 9.4, 9.3 us, forty 24.7,
           18.4, 18.4, sixteen 11.8, 11.8, 17.5, where a second round of clusters begins).  Against two launches, 32 + 8 heads of
           128, at 1024, 2048, 4096, 8192 and 16384 keys: bf16 6.5 / 8.8, 7.8 / 9.9, 9.5 / 9.7, 12.9 / 12.3, 19.1 / 15.4 us; e4m3
           7.5 / 8.9, 8.6 / 9.7, 10.7 / 9.5, 14.8 / 12.2, 22.8 / 15.3.  (Heads of 256 would do better without: bf16 12.8 / 11.3,
           15.2 / 12.2, 19.3 / 12.4.) */
        p.in_clusters = true;
        while (p.splits < 16u && (uint64_t)p.splits * 64u < keys && ctas * p.splits * 2u <= (uint64_t)sms * 5u / 4u) p.splits *= 2u;
        return p;
    }
    /* no CTA below a tile for each of its warps */
    const uint64_t most = (keys + 383u) / 384u, want = (uint64_t)sms > ctas ? (uint64_t)sms / ctas : 1u;
    p.splits = (uint32_t)(want < most ? want : most);
    p.cells = p.splits > 1u ? (uint64_t)p.splits * T * n_q : 0u;
    return p;
}

cudaError_t launch_kv_attention(cudaStream_t st, int elem, uint32_t head_dim, const KvAttention &a, const KvPlan &p, int sms) {
    if (p.many) return launch_kv_many(st, elem, head_dim, a, sms);
    if (elem == kKvE4m3) return head_dim == 64u ? launch_all<64, kKvE4m3>(st, a, p) : head_dim == 128u ? launch_all<128, kKvE4m3>(st, a, p) : launch_all<256, kKvE4m3>(st, a, p);
    return head_dim == 64u ? launch_all<64, kKvBf16>(st, a, p) : head_dim == 128u ? launch_all<128, kKvBf16>(st, a, p) : launch_all<256, kKvBf16>(st, a, p);
}

void configure_kv_kernels() { configure_kv_many(); configure_few<64>(); configure_few<128>(); configure_few<256>(); }

}  // namespace nwc
