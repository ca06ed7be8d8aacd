// Attention over a paged cache held in 4 bits, for sequences of different lengths.
#include "attention_kv4_stream.h"

namespace mynn {

int paged_kv_check(const char *who, const PagedKv &c, int page_rows, int kv_bits, int group, int D);
int paged_shift(int page_rows);

// One wave for a query row of a head: 64 keys at a time, a key a lane; then a lane's dims over those keys.
template <typename T, int D> __global__ __launch_bounds__(64) void attn_kv4_row_kernel(Kv4Args a, int group) {
    __shared__ float q_s[D], p_s[64];
    __shared__ size_t r_s[64];
    const int lane = threadIdx.x, i = blockIdx.x % a.Sq, head = blockIdx.x / a.Sq, b = blockIdx.y;
    const int h = head / (a.Hq / a.c.Hkv), groups = D / group;
    const PagedSeq seq(a.c, b, a.Sq);
    const int bound = seq.bound(i, a.causal);
    const size_t line = (((size_t)b * a.Hq + head) * a.Sq + i) * D;
    for (int d = lane; d < D; d += 64) q_s[d] = Elem<T>::ld((const T *)a.q, line + d);
    float m = -INFINITY, l = 0.f, o[D / 64] = {};
    for (int k0 = 0; k0 < bound; k0 += 64) {
        __syncthreads();
        const int key = k0 + lane, page = key < bound ? paged_page(a.c, b, key) : -1;
        const size_t r = page >= 0 ? paged_row(a.c, page, h, key) : 0;
        float s = -INFINITY;
        if (page >= 0) {
            s = 0.f;
            for (int g = 0; g < groups; g++) {
                float x = 0.f;
                const float z = (float)(a.c.k_zero[r * groups + g] & 15);
                for (int d = g * group; d < (g + 1) * group; d++) {
                    const uint32_t w = ((const uint8_t *)a.c.k)[r * (D / 2) + d / 2];
                    x = fmaf(q_s[d], (float)(d & 1 ? w >> 4 : w & 15u) - z, x);
                }
                s = fmaf(x, Elem<T>::ld((const T *)a.c.k_scale, r * groups + g), s);
            }
            s *= a.scale;
        }
        const float mn = fmaxf(m, wave_max(s)), ref = mn == -INFINITY ? 0.f : mn;
        const float p = page >= 0 ? expf(s - ref) : 0.f, corr = expf(m - ref);
        m = mn;
        l = l * corr + wave_sum(p);
        p_s[lane] = p;
        r_s[lane] = page >= 0 ? r : ~(size_t)0;
        __syncthreads();
        for (int e = 0; e < D / 64; e++) {
            const int d = lane + 64 * e, g = d / group;
            float x = 0.f;
            for (int k = 0; k < 64; k++) {
                const size_t rk = r_s[k];
                if (rk == ~(size_t)0) continue;
                const uint32_t w = ((const uint8_t *)a.c.v)[rk * (D / 2) + d / 2];
                const float z = (float)(a.c.v_zero[rk * groups + g] & 15), sc = Elem<T>::ld((const T *)a.c.v_scale, rk * groups + g);
                x = fmaf(p_s[k], ((float)(d & 1 ? w >> 4 : w & 15u) - z) * sc, x);
            }
            o[e] = o[e] * corr + x;
        }
    }
    for (int e = 0; e < D / 64; e++) Elem<T>::st((T *)a.out, line + lane + 64 * e, l == 0.f ? 0.f : o[e] / l);
}

static int kv4_cus() {
    static int cus = 0;
    if (!cus) {
        int dev = 0, n = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) {
            (void)hipGetLastError();
            n = 256;
        }
        cus = n;
    }
    return cus;
}
static bool kv4_few_rows(int Hq, int Hkv, int Sq) { return (long)(Hq / Hkv) * Sq <= 16; }
// workgroups of the form for few rows: as many as run at once, no more than there can be units
static int kv4_stream_grid(int B, int Hkv, long rows) {
    const long units = (long)B * Hkv * ((rows + kKv4Unit - 1) / kKv4Unit), most = 2l * kv4_cus();
    return (int)(units < most ? units : most);
}

template <typename T, int D, int NG> static int kv4_stream_go(const Kv4Args &a, hipStream_t s) {
    const int R = a.Hq / a.c.Hkv * a.Sq, tile = 32 * (D / 2 + 16), wave = tile > R * D * 4 ? tile : R * D * 4;
    MYNN_LAUNCH((attn_kv4_stream_kernel<T, D, NG>), dim3(a.grid), dim3(kKv4Waves * 64), kKv4Waves * (wave + 128), s, a);
    if (const int rc = launch_status("attn_kv4_stream_kernel")) return rc;
    if (a.grid == a.B * a.c.Hkv && a.c.pages_per_seq << a.c.page_shift <= kKv4Unit) return 0;  // (a unit each: nothing is shared)
    MYNN_LAUNCH((attn_kv4_join_kernel<T, D>), dim3(a.B * a.c.Hkv), dim3(256), 0, s, a);
    return launch_status("attn_kv4_join_kernel");
}

}  // namespace mynn

using namespace mynn;

extern "C" size_t mynn_attention_paged_int4_workspace_bytes(int B, int Sq, int pages_per_seq, int page_rows, int num_q_heads, int num_kv_heads, int head_dim) {
    if (B <= 0 || Sq <= 0 || pages_per_seq <= 0 || page_rows <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || !kv4_few_rows(num_q_heads, num_kv_heads, Sq)) return 0;
    const size_t R = (size_t)(num_q_heads / num_kv_heads) * Sq;
    return 2 * (size_t)kv4_stream_grid(B, num_kv_heads, (long)pages_per_seq * page_rows) * R * (head_dim + 4) * sizeof(float);
}

extern "C" int mynn_attention_paged_int4(void *out, const void *Q, const uint8_t *k_pool, const uint8_t *v_pool, const void *k_scale_pool, const void *v_scale_pool,
                                         const uint8_t *k_zero_pool, const uint8_t *v_zero_pool, const int32_t *page_table, int n_pages, int pages_per_seq, int page_rows,
                                         float scale, int is_causal, int B, int Sq, const int32_t *past_lens, const int32_t *new_lens, int num_q_heads, int num_kv_heads,
                                         int head_dim, int dtype, int group, void *workspace, size_t workspace_bytes, int32_t *counters, mynn_stream s) {
    const char *who = "attention_paged_int4";
    MYNN_REQUIRE(out && Q && aligned16(out) && aligned16(Q), MYNN_ERR_INVALID, "%s: null or unaligned operand", who);
    MYNN_REQUIRE(B > 0 && Sq > 0 && num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0, MYNN_ERR_INVALID, "%s: B=%d Sq=%d heads %d/%d", who, B, Sq,
                 num_q_heads, num_kv_heads);
    Kv4Args a{{(void *)k_pool, (void *)v_pool, (void *)k_scale_pool, (void *)v_scale_pool, (uint8_t *)k_zero_pool, (uint8_t *)v_zero_pool, page_table, past_lens, new_lens,
               n_pages, pages_per_seq, 0, num_kv_heads},
              out, Q, scale, is_causal, B, Sq, num_q_heads, nullptr, nullptr, nullptr, 0};
    if (const int rc = paged_kv_check(who, a.c, page_rows, 4, group, head_dim)) return rc;
    a.c.page_shift = paged_shift(page_rows);
    MYNN_REQUIRE((long)num_q_heads * Sq < 1l << 31 && B <= 65535, MYNN_ERR_UNSUPPORTED, "%s: B=%d Sq=%d heads %d", who, B, Sq, num_q_heads);
    if (kv4_few_rows(num_q_heads, num_kv_heads, Sq)) {
        const size_t need = mynn_attention_paged_int4_workspace_bytes(B, Sq, pages_per_seq, page_rows, num_q_heads, num_kv_heads, head_dim);
        MYNN_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need), MYNN_ERR_INVALID, "%s: %zu bytes of workspace, %zu needed", who,
                     workspace_bytes, need);
        MYNN_REQUIRE((long)B * num_kv_heads * (((long)pages_per_seq * page_rows + kKv4Unit - 1) / kKv4Unit) < 1l << 30, MYNN_ERR_UNSUPPORTED,
                     "%s: %d sequences of %d heads of %ld rows", who, B, num_kv_heads, (long)pages_per_seq * page_rows);
        a.grid = kv4_stream_grid(B, num_kv_heads, (long)pages_per_seq * page_rows);
        const size_t R = (size_t)(num_q_heads / num_kv_heads) * Sq;
        a.part_o = (float *)workspace;
        a.part_ml = a.part_o + 2 * (size_t)a.grid * R * head_dim;
        a.counters = counters;
        return dispatch_dtype16(dtype, [&](auto *t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (head_dim == 64) return group == 64 ? kv4_stream_go<T, 64, 1>(a, as_stream(s)) : kv4_stream_go<T, 64, 2>(a, as_stream(s));
            return group == 128 ? kv4_stream_go<T, 128, 1>(a, as_stream(s)) : group == 64 ? kv4_stream_go<T, 128, 2>(a, as_stream(s)) : kv4_stream_go<T, 128, 4>(a, as_stream(s));
        });
    }
    return dispatch_dtype16(dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const dim3 grid(num_q_heads * Sq, B);
        if (head_dim == 64) MYNN_LAUNCH((attn_kv4_row_kernel<T, 64>), grid, dim3(64), 0, as_stream(s), a, group);
        else MYNN_LAUNCH((attn_kv4_row_kernel<T, 128>), grid, dim3(64), 0, as_stream(s), a, group);
        return launch_status("attn_kv4_row_kernel");
    });
}
