// Attention over a paged cache held in 4 bits, for sequences of different lengths.
#include "attention_kv4_stream.h"
#include "attention_kv4_tile.h"

namespace mynn {

int paged_kv_check(const char *who, const PagedKv &c, int page_rows, int kv_bits, int group, int D);
int paged_shift(int page_rows);

template <int N> using Int = std::integral_constant<int, N>;

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

// Rows of a workgroup of the form for many rows, and the ranges that its keys come in where blocks of rows leave the device idle.
struct Kv4TilePlan {
    int rows, blocks, ranges;
};
static Kv4TilePlan kv4_tile_plan(int B, int Sq, int Hq, int Hkv, long rows) {
    const long R = (long)(Hq / Hkv) * Sq;
    Kv4TilePlan p;
    p.rows = R <= 64 ? 64 : 128;
    p.blocks = (int)((R + p.rows - 1) / p.rows);
    const long wgs = (long)B * Hkv * p.blocks, most = (rows + 255) / 256, want = 2l * kv4_cus() / wgs;
    p.ranges = (int)(want < 1 ? 1 : want > most ? most : want);
    return p;
}

template <typename T, int D, int NG, int QW, int KW> static int kv4_tile_launch(const Kv4Args &a, const Kv4TilePlan &p, hipStream_t s) {
    using Block = Kv4Block<D, NG, QW, KW, 64>;
    static bool set = false;
    if (!set && Block::LDS > 64 * 1024) {
        MYNN_HIP(hipFuncSetAttribute((const void *)attn_kv4_tile_kernel<T, D, NG, QW, KW, 64>, hipFuncAttributeMaxDynamicSharedMemorySize, Block::LDS));
        set = true;
    }
    MYNN_LAUNCH((attn_kv4_tile_kernel<T, D, NG, QW, KW, 64>), dim3(a.B * a.c.Hkv, p.blocks, p.ranges), dim3(Block::THREADS), Block::LDS, s, a);
    return launch_status("attn_kv4_tile_kernel");
}
template <typename T, int D, int NG> static int kv4_tile_go(const Kv4Args &a, const Kv4TilePlan &p, hipStream_t s) {
    const int rc = p.rows == 64 ? kv4_tile_launch<T, D, NG, 2, 2>(a, p, s) : kv4_tile_launch<T, D, NG, 4, 1>(a, p, s);
    if (rc || p.ranges == 1) return rc;
    const size_t threads = (size_t)a.B * a.Hq * a.Sq * (D / 4);
    MYNN_LAUNCH((attn_kv4_ranges_kernel<T, D>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, a, p.ranges, p.rows);
    return launch_status("attn_kv4_ranges_kernel");
}

}  // namespace mynn

using namespace mynn;

extern "C" size_t mynn_attention_paged_int4_workspace_bytes(int B, int Sq, int pages_per_seq, int page_rows, int num_q_heads, int num_kv_heads, int head_dim) {
    if (B <= 0 || Sq <= 0 || pages_per_seq <= 0 || page_rows <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads) return 0;
    const size_t R = (size_t)(num_q_heads / num_kv_heads) * Sq;
    if (!kv4_few_rows(num_q_heads, num_kv_heads, Sq)) {
        const int ranges = kv4_tile_plan(B, Sq, num_q_heads, num_kv_heads, (long)pages_per_seq * page_rows).ranges;
        return ranges == 1 ? 0 : (size_t)ranges * B * num_kv_heads * R * (head_dim + 4) * sizeof(float);
    }
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
    MYNN_REQUIRE((long)num_q_heads * Sq < 1l << 30 && (long)B * num_kv_heads < 1l << 30, MYNN_ERR_UNSUPPORTED, "%s: B=%d Sq=%d heads %d", who, B, Sq, num_q_heads);
    const long rows = (long)pages_per_seq * page_rows;
    const size_t need = mynn_attention_paged_int4_workspace_bytes(B, Sq, pages_per_seq, page_rows, num_q_heads, num_kv_heads, head_dim);
    MYNN_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need), MYNN_ERR_INVALID, "%s: %zu bytes of workspace, %zu needed", who, workspace_bytes,
                 need);
    const size_t R = (size_t)(num_q_heads / num_kv_heads) * Sq;
    a.part_o = (float *)workspace;
    auto pick = [&](auto &&go) {
        return dispatch_dtype16(dtype, [&](auto *t) {
            if (head_dim == 64) return group == 64 ? go(t, Int<64>{}, Int<1>{}) : go(t, Int<64>{}, Int<2>{});
            return group == 128 ? go(t, Int<128>{}, Int<1>{}) : group == 64 ? go(t, Int<128>{}, Int<2>{}) : go(t, Int<128>{}, Int<4>{});
        });
    };
    if (kv4_few_rows(num_q_heads, num_kv_heads, Sq)) {
        MYNN_REQUIRE((long)B * num_kv_heads * ((rows + kKv4Unit - 1) / kKv4Unit) < 1l << 30, MYNN_ERR_UNSUPPORTED, "%s: %d sequences of %d heads of %ld rows", who, B, num_kv_heads,
                     rows);
        a.grid = kv4_stream_grid(B, num_kv_heads, rows);
        a.part_ml = a.part_o + 2 * (size_t)a.grid * R * head_dim;
        a.counters = counters;
        return pick([&](auto *t, auto d, auto n) { return kv4_stream_go<std::remove_pointer_t<decltype(t)>, decltype(d)::value, decltype(n)::value>(a, as_stream(s)); });
    }
    const Kv4TilePlan plan = kv4_tile_plan(B, Sq, num_q_heads, num_kv_heads, rows);
    MYNN_REQUIRE(plan.blocks <= 65535 && plan.ranges <= 65535, MYNN_ERR_UNSUPPORTED, "%s: Sq=%d heads %d/%d", who, Sq, num_q_heads, num_kv_heads);
    a.part_ml = a.part_o + (size_t)plan.ranges * B * num_kv_heads * R * head_dim;
    return pick([&](auto *t, auto d, auto n) { return kv4_tile_go<std::remove_pointer_t<decltype(t)>, decltype(d)::value, decltype(n)::value>(a, plan, as_stream(s)); });
}
