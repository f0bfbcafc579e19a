// Attention of new tokens over a paged key/value cache.
//
// out[t,h] = sum_j p_j v_j, p = softmax_j(scale q.k_j) over the keys token t sees, in one pass over the keys with a running maximum m
// and sum l: a tile's scores s give m' = max(m, s), p = exp(s - m'), l = l exp(m - m') + sum p, o = o exp(m - m') + sum p v.
// A wave per (token, query head): a lane scores one key of a tile of 64, then owns channels lane, lane + 64, .. of the output.
#include "decode_common.h"

namespace ttsamd {
namespace {

struct AttArgs {
    ttsamd_paged_attention_args a;
    ttsamd_paged_kv c;
    ttsamd_paged_batch b;
    FastDiv by_page;
};

template <class T> __global__ __launch_bounds__(64) void attend_rows(AttArgs g)
{
    __shared__ float sq[256], sp[64];
    __shared__ int64_t sv[64];
    const Sequence s = sequence_of(g.b, g.a.tokens, g.c.page_size, blockIdx.z);
    const int h = blockIdx.y, hk = h / (g.a.q_heads / g.c.kv_heads), lane = threadIdx.x, d = g.c.head_dim;
    for (int i = blockIdx.x; i < s.n; i += gridDim.x) {
        const int64_t token = s.start + i;
        const T *q = (const T *)g.a.q + token * g.a.q_tstride + h * g.a.q_hstride;
        __syncthreads();
        for (int e = lane; e < d; e += 64) sq[e] = to_f(q[e]);
        __syncthreads();
        const int pos = s.len - s.n + i;
        const auto [begin, end] = seen_by(s, pos, g.a.causal, g.a.window);
        float m = -INFINITY, l = 0.f, o[4] = {};
        for (int base = begin; base < end; base += 64) {
            const int j = base + lane;
            float w = -INFINITY;
            int64_t at = -1;
            if (j < end) {
                int row;
                const int64_t page = page_of(g.b, g.by_page, g.c.pages, blockIdx.z, j, row);
                if (page >= 0) {
                    const T *k = (const T *)g.c.k + page * g.c.k_page + hk * g.c.k_head + row * g.c.k_row;
                    at = page * g.c.v_page + hk * g.c.v_head + row * g.c.v_row;
                    w = 0.f;
                    for (int e = 0; e < d; ++e) w = fmaf(sq[e], to_f(k[e]), w);
                    w *= g.a.scale;
                }
            }
            float top = w;
            for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
            const float m2 = fmaxf(m, top);
            const float p = at < 0 || m2 == -INFINITY ? 0.f : expf(w - m2), fade = m2 == -INFINITY ? 1.f : expf(m - m2);
            float sum = p;
            for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
            l = l * fade + sum, m = m2;
            __syncthreads();
            sp[lane] = p, sv[lane] = at;
            __syncthreads();
            for (int x = 0; x < 4; ++x) o[x] *= fade;
            for (int r = 0; r < 64; ++r) {
                if (sv[r] < 0) continue;
                const T *v = (const T *)g.c.v + sv[r];
                for (int x = 0; x < 4; ++x)
                    if (lane + 64 * x < d) o[x] = fmaf(sp[r], to_f(v[lane + 64 * x]), o[x]);
            }
        }
        T *out = (T *)g.a.out + token * g.a.o_tstride + h * g.a.o_hstride;
        for (int x = 0; x < 4; ++x)
            if (lane + 64 * x < d) out[lane + 64 * x] = (T)(l > 0.f ? o[x] / l : l == 0.f ? 0.f : o[x] + l);
    }
}

}  // namespace
}  // namespace ttsamd

extern "C" size_t ttsamd_paged_attention_workspace_bytes(const ttsamd_paged_attention_args *, const ttsamd_paged_kv *, const ttsamd_paged_batch *)
{
    return 0;
}

extern "C" int ttsamd_paged_attention(const ttsamd_paged_attention_args *a, const ttsamd_paged_kv *cache, const ttsamd_paged_batch *batch,
                                      void *, size_t, void *stream)
{
    using namespace ttsamd;
    TTSAMD_CHECK_ARG(a, "paged_attention: arguments are NULL");
    if (int rc = check_paged_kv("paged_attention", cache)) return rc;
    if (int rc = check_paged_batch("paged_attention", batch, a->tokens)) return rc;
    TTSAMD_CHECK_ARG(a->q_heads > 0 && a->q_heads % cache->kv_heads == 0, "paged_attention: %d query heads over %d key heads", a->q_heads,
                     cache->kv_heads);
    TTSAMD_CHECK_ARG(a->window >= 0, "paged_attention: window %d", a->window);
    if (a->tokens == 0 || batch->batch == 0) return TTSAMD_OK;
    TTSAMD_CHECK_ARG(a->q && a->out, "paged_attention: a tensor is NULL");
    const int per = 16 / elem_bytes(cache->dtype);
    TTSAMD_CHECK_ARG((((uintptr_t)a->q | (uintptr_t)a->out) & 15) == 0 && a->q_tstride % per == 0 && a->q_hstride % per == 0 &&
                         a->o_tstride % per == 0 && a->o_hstride % per == 0,
                     "paged_attention: q and out start and stride at multiples of 16 bytes");
    if (a->q_heads > 65535) {
        set_error("paged_attention: %d query heads (up to 65535)", a->q_heads);
        return TTSAMD_ERR_UNSUPPORTED;
    }
    AttArgs g{*a, *cache, *batch, fast_div(cache->page_size)};
    const dim3 grid(batch->max_new < 1 ? 1 : batch->max_new, a->q_heads, batch->batch);
    hipStream_t st = as_stream(stream);
    if (cache->dtype == TTSAMD_F32) attend_rows<float><<<grid, 64, 0, st>>>(g);
    else if (cache->dtype == TTSAMD_F16) attend_rows<_Float16><<<grid, 64, 0, st>>>(g);
    else attend_rows<__bf16><<<grid, 64, 0, st>>>(g);
    TTSAMD_LAUNCH_CHECK();
    return TTSAMD_OK;
}
