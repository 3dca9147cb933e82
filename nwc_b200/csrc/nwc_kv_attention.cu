/* Attention of one or many tokens over a cache of nwc_kv.h: o_t = sum over the positions p that token t sees of
 * softmax_p(scale q_t . k_p) v_p, grouped heads; zeros where a token sees nothing.
 *
 * What token t (position own = pos + t, or pos + depth[t] with a draft tree) sees:
 *   p < pos + T with p <= own (no tree) or p < pos or bit p - pos of visible[t] (tree); and, with a window and for p that are
 *   not drafted, p < sinks or p > own - window.
 */
#include "nwc_kv.h"
#include "nwc_launch.h"

namespace nwc {

__device__ __forceinline__ void kv_dependency_sync() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

/* The plain kernel: one CTA per token and query head, its warps take the visible positions in turn, lanes own head_dim / 32
   numbers each; online softmax in fp32. */
template <int VPL, int ELEM>
__global__ void __launch_bounds__(128) kv_attention_plain_kernel(const KvAttention a) {
    constexpr uint32_t HD = 32u * VPL, kWarps = 4;
    __shared__ float part_max[kWarps], part_den[kWarps], part_acc[kWarps][HD];
    const uint32_t t = blockIdx.x, head = blockIdx.y, kvh = head / (a.n_q / a.c.n_kv), lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, d0 = lane * VPL;
    kv_dependency_sync();
    const int32_t pos = *a.pos;
    const uint32_t limit = a.c.window ? 0x7FFFFFFFu : a.c.capacity;
    if (pos < 0 || (uint64_t)pos + a.T > limit) { if (threadIdx.x == 0) atomicOr(a.status, kKvStatusPosition); return; }
    const KvSpan span = kv_span(pos, a.T, a.c.window, a.c.sinks);
    const uint32_t own = a.depth ? (uint32_t)(pos + a.depth[t]) : (uint32_t)pos + t, words = (a.T + 31u) / 32u;
    float q[VPL], acc[VPL], m = -INFINITY, den = 0.f;
    const uint16_t *qp = a.q + (uint64_t)t * a.ldq + (uint64_t)head * HD + d0;
#pragma unroll
    for (int j = 0; j < VPL; j++) { q[j] = __uint_as_float((uint32_t)qp[j] << 16) * a.scale; acc[j] = 0.f; }
    for (uint32_t i = warp; i < span.count; i += kWarps) {
        const uint32_t p = i < span.lead ? i : span.first + (i - span.lead);
        bool sees = !a.c.window || p < a.c.sinks || p + a.c.window > own;
        if (!a.visible) sees = sees && p <= own;
        else if (p >= (uint32_t)pos) { const uint32_t j = p - (uint32_t)pos; sees = (a.visible[(uint64_t)t * words + (j >> 5)] >> (j & 31u)) & 1u; }
        if (!sees) continue;
        const uint64_t cell = (uint64_t)kvh * a.c.capacity + kv_slot(p, a.c.capacity, a.c.window, a.c.sinks);
        float k[VPL], v[VPL];
        if (ELEM == kKvBf16) {
            const uint16_t *kp = reinterpret_cast<const uint16_t *>(a.c.k) + cell * HD + d0, *vp = reinterpret_cast<const uint16_t *>(a.c.v) + cell * HD + d0;
#pragma unroll
            for (int j = 0; j < VPL; j++) { k[j] = __uint_as_float((uint32_t)kp[j] << 16); v[j] = __uint_as_float((uint32_t)vp[j] << 16); }
        } else {
            const uint32_t ku = kv_unit2(a.c.k_exp[cell]), vu = kv_unit2(a.c.v_exp[cell]);
            const uint8_t *kp = a.c.k + cell * HD + d0, *vp = a.c.v + cell * HD + d0;
#pragma unroll
            for (int j = 0; j < VPL; j += 2) {
                uint32_t kw, vw, none;
                kv_values4((uint32_t)kp[j] | ((uint32_t)kp[j + 1] << 8), ku, kw, none);
                kv_values4((uint32_t)vp[j] | ((uint32_t)vp[j + 1] << 8), vu, vw, none);
                k[j] = __uint_as_float(kw << 16); k[j + 1] = __uint_as_float(kw & 0xFFFF0000u);
                v[j] = __uint_as_float(vw << 16); v[j + 1] = __uint_as_float(vw & 0xFFFF0000u);
            }
        }
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < VPL; j++) s = fmaf(q[j], k[j], s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const float m_new = fmaxf(m, s), corr = m_new == -INFINITY ? 1.f : exp2f(m - m_new), w = m_new == -INFINITY ? 0.f : exp2f(s - m_new);
        den = den * corr + w;
#pragma unroll
        for (int j = 0; j < VPL; j++) acc[j] = fmaf(w, v[j], acc[j] * corr);
        m = m_new;
    }
    if (lane == 0) { part_max[warp] = m; part_den[warp] = den; }
#pragma unroll
    for (int j = 0; j < VPL; j++) part_acc[warp][d0 + j] = acc[j];
    __syncthreads();
    float top = part_max[0];
    for (uint32_t w = 1; w < kWarps; w++) top = fmaxf(top, part_max[w]);
    for (uint32_t d = threadIdx.x; d < HD; d += blockDim.x) {
        float total = 0.f, o = 0.f;
        for (uint32_t w = 0; w < kWarps; w++) {
            const float f = top == -INFINITY ? 0.f : exp2f(part_max[w] - top);
            total = fmaf(part_den[w], f, total); o = fmaf(part_acc[w][d], f, o);
        }
        const float r = total == 0.f ? 0.f : o / total;
        a.out[((uint64_t)t * a.n_q + head) * HD + d] = __bfloat16_as_ushort(__float2bfloat16_rn(r));
    }
}

template <int VPL>
static cudaError_t launch_plain(cudaStream_t st, int elem, const KvAttention &a) {
    const dim3 grid(a.T, a.n_q);
    if (elem == kKvE4m3) kv_attention_plain_kernel<VPL, kKvE4m3><<<grid, 128, 0, st>>>(a);
    else kv_attention_plain_kernel<VPL, kKvBf16><<<grid, 128, 0, st>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_kv_attention(cudaStream_t st, int elem, uint32_t head_dim, const KvAttention &a) {
    return head_dim == 64u ? launch_plain<2>(st, elem, a) : head_dim == 128u ? launch_plain<4>(st, elem, a) : launch_plain<8>(st, elem, a);
}

}  // namespace nwc
