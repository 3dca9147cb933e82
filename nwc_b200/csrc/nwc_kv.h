/* The key/value cache of nwc_kv_*: where a position lives, which positions a token sees, and how a quantised row is held.
 *
 * Slots.  Without a window position p lives in slot p.  With one, the cache is `sinks` fixed slots followed by a ring of
 * capacity - sinks slots: positions from `sinks` on take the ring's slots in turn, so a session of any length fits.
 *
 * Quantised rows.  One row (head_dim numbers of one head) = e4m3 codes and one byte b: value = code * 2^(b - 127) with the
 * smallest exponent that keeps the row's largest magnitude within 448 * 2^(b - 127).  e4m3 is a floating-point type, so its
 * relative error does not depend on where in its range a number lies: a finer scale than a power of two would buy nothing but
 * the distance to the subnormal range, while multiplying by a power of two is exact - quantising rounds once (by at most 2^-4
 * relative, and below 2^-6 of the unit by 2^-10 units), reading back not at all.
 */
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include "../../include/nwc_ops.h"

namespace nwc {

constexpr int kKvBf16 = 0, kKvE4m3 = 1;
constexpr int kKvStatusPosition = 1, kKvStatusNotFinite = 2, kKvStatusPath = 4, kKvStatusWait = 8;      /* bits of the status word */

/* One layer of a cache. */
struct KvLayer {
    uint8_t *k, *v;             /* [n_kv][capacity][head_dim], bf16 or codes */
    uint8_t *k_exp, *v_exp;     /* [n_kv][capacity], e4m3 only */
    uint32_t n_kv, capacity, window, sinks;
};

__host__ __device__ __forceinline__ uint32_t kv_slot(uint32_t p, uint32_t capacity, uint32_t window, uint32_t sinks) {
    return !window || p < sinks ? p : sinks + (p - sinks) % (capacity - sinks);
}

/* The keys a call visits, as one list: the sinks that the window does not reach (`lead` of them, positions 0 .. lead - 1),
   then positions `first` .. pos + T - 1. */
struct KvSpan { uint32_t lead, first, count; };
__host__ __device__ __forceinline__ KvSpan kv_span(uint32_t pos, uint32_t T, uint32_t window, uint32_t sinks) {
    KvSpan s;
    s.first = window && pos + 1u > window ? pos + 1u - window : 0u;
    s.lead = sinks < s.first ? sinks : s.first;
    s.count = s.lead + (pos + T - s.first);
    return s;
}

/* 2^(b - 127) in fp32 */
__device__ __forceinline__ float kv_unit(uint32_t b) { return __uint_as_float(b ? b << 23 : 1u << 22); }

/* four e4m3 codes -> two bf16x2 words with the values times 2^-120: the code's exponent and mantissa bits are moved into the
   bf16 fields as they are (e4m3 subnormals become bf16 subnormals of the same value), so the bias difference 127 - 7 is all
   that is left to multiply by.  The NaN codes 0x7F / 0xFF become 480 here; kv_has_nan() finds them. */
__device__ __forceinline__ void kv_spread(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t a = __byte_perm(w, 0u, 0x1404), b = __byte_perm(w, 0u, 0x3424);
    lo = ((a >> 4) & 0x07F007F0u) | (a & 0x80008000u);
    hi = ((b >> 4) & 0x07F007F0u) | (b & 0x80008000u);
}
__device__ __forceinline__ bool kv_has_nan(uint32_t w) { return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0u; }
__device__ __forceinline__ uint32_t kv_mul2(uint32_t a, uint32_t b) { uint32_t d; asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b)); return d; }
constexpr uint32_t kTwoTo120 = 0x7B807B80u;                              /* bf16 pair */
/* 2^(b - 127) as a bf16 pair (b = 0: the subnormal 2^-127) */
__device__ __forceinline__ uint32_t kv_unit2(uint32_t b) { const uint32_t h = b ? b << 7 : 0x40u; return h | (h << 16); }
/* four codes -> four bf16 values code * 2^(b - 127); exact where the value is a normal bf16 number */
__device__ __forceinline__ void kv_values4(uint32_t w, uint32_t unit2, uint32_t &lo, uint32_t &hi) {
    kv_spread(w, lo, hi);
    lo = kv_mul2(kv_mul2(lo, kTwoTo120), unit2);
    hi = kv_mul2(kv_mul2(hi, kTwoTo120), unit2);
    if (kv_has_nan(w)) {
        if ((w & 0x7Fu) == 0x7Fu) lo |= 0x00007FC0u;
        if ((w & 0x7F00u) == 0x7F00u) lo |= 0x7FC00000u;
        if ((w & 0x7F0000u) == 0x7F0000u) hi |= 0x00007FC0u;
        if ((w & 0x7F000000u) == 0x7F000000u) hi |= 0x7FC00000u;
    }
}

/* Arguments of the attention kernels. */
struct KvAttention {
    KvLayer c;
    const uint16_t *q;           /* bf16 rows of n_q * head_dim, ldq apart */
    uint64_t ldq;
    uint32_t T, n_q;
    const int32_t *pos;          /* device */
    const uint32_t *visible;     /* [T][(T + 31) / 32] or null */
    const int32_t *depth;        /* [T] or null */
    float scale;                 /* softmax scale times log2(e) */
    uint16_t *out;               /* bf16 [T][n_q * head_dim] */
    int *status;
    /* Where a row's keys are divided over `splits` CTAs, each leaves its share here, fp32: the unnormalised outputs, and running
       maximum (log2) and sum.  Few rows: part_o [splits][T * n_q][head_dim], part_ml [splits][T * n_q][2].  Many: part_o
       [splits][units][2][head_dim / 4][128][4], part_ml [splits][units][2][128][2]. */
    float *part_o, *part_ml;
    uint32_t splits;
    uint32_t layer, layers;      /* which layer of how many `c` is */
    uint32_t pairs;              /* many: units of two row tiles; those behind them have one */
};
/* How a call is divided.  It goes by sizes that the host knows (a captured call is replayed at other positions): the most
   keys that the cache can show, not the position. */
constexpr uint32_t kKvShortKeys = 4096;
struct KvPlan {
    uint32_t splits;             /* CTAs that divide the keys of one head's rows */
    bool in_clusters, many;      /* many: the tensor-memory kernel of nwc_kv_many.cu */
    uint64_t cells;              /* rows of shares in the workspace, head_dim + 2 fp32 numbers each */
};
KvPlan kv_attention_plan(int elem, uint32_t head_dim, uint32_t n_kv, uint32_t capacity, uint32_t window, uint32_t sinks, uint32_t T, uint32_t n_q, int sms);
cudaError_t launch_kv_attention(cudaStream_t st, int elem, uint32_t head_dim, const KvAttention &a, const KvPlan &plan, int sms);
cudaError_t launch_kv_many(cudaStream_t st, int elem, uint32_t head_dim, const KvAttention &a, int sms);
void configure_kv_many();
cudaError_t launch_kv_wait_probe(cudaStream_t st, int *status);
void configure_kv_kernels();                 /* per-device shared-memory opt-ins */
int read_kv_status(bool clear);              /* 0, or 2 when a bounded wait gave up */

}  // namespace nwc
