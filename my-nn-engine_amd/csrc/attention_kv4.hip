// Attention over a paged cache held in 4 bits, for sequences of different lengths.
#include <algorithm>

#include "attention_kv4_stream.h"
#include "attention_kv4_tile.h"

namespace mynn {

int paged_kv_check(const char *who, const PagedKv &c, int page_rows, int kv_bits, int group, int D);
int paged_shift(int page_rows);

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
// How often the rows are put side by side: as 16 columns have room for them.  (Four groups of columns a row: twice at the most, the tile of 64 keys does not fit the registers.)
static int kv4_fold(long rows, int groups) { return rows <= 4 && groups < 4 ? 4 : rows <= 8 ? 2 : 1; }
// Waves that share a (sequence, kv head)'s keys step by step.  Four; one where there is a (sequence, kv head) for each wave, or fewer and few keys: what a workgroup
// waits for at its ends -- lengths, pages, the first codes, the others' results -- another's work fills then (32 / 8 heads of 128, one token of 256 sequences of 64 keys 24 us and,
// one wave each, 13, of 512 47 and 38, of 8192 587 and 568; 128 of 256 17 and 15, of up to 2048 62 and 64; 64 of 128 10.4 and 8.8, of 256 11 and 13).  More than 8 rows keep four: the join by a single wave would have 16 pairs of columns a lane.
static int kv4_waves(long pairs, long R, long rows) {
    const long cus = kv4_cus();
    return R <= 8 && (pairs >= 8 * cus || (pairs >= 4 * cus && rows <= 512) || (pairs >= 2 * cus && rows <= 128)) ? 1 : 4;
}
static int kv4_unit(int fold, int waves) { return waves * (fold == 4 ? kKv4Keys<4> : kKv4Keys<1>); }
// workgroups of the form for few rows: as many as run at once, no more than there can be units, or than there are counters
static int kv4_stream_grid(long pairs, int unit, int waves, long rows) {
    const long units = pairs * ((rows + unit - 1) / unit), all = std::min(8l / waves * kv4_cus(), (long)MYNN_PAGED_INT4_COUNTERS);
    if (waves == 1) return (int)std::min(all, pairs);
    // Two a CU; where that makes more than 32 parts of a (sequence, kv head), fewer: their join is on one CU (one sequence of 32768 keys, 8 kv heads of 128: with 64 parts each
    // 24 us, with 32 20, with 16 23).
    return (int)std::min(units, std::min(all, std::max(32 * pairs, all / 4)));
}

// Rows of a workgroup, and up to how many ranges of keys its rows' keys come in (two workgroups a CU run at once; Kv4TilePlan::ranges makes twice that at the most, how many
// of them a block takes is found on the device).  R: rows of a kv head, rows: those of a sequence's pages in the table, which is all that the host knows of lengths (here and in
// kv4_waves).  The figures are of tables as wide as the longest sequence.  A table far wider than that has calls take the forms for long caches: over 8192 rows prompts of
// 100 rows 15 us for 12, of 1200 59 for 40, 3 x 333 36 for 19, 8 x 64 tokens behind 1000 rows 39 for 34, 64 sequences of 128 keys 8.8 for 8.3.
static Kv4TilePlan kv4_tile_plan(int B, int Sq, int Hq, int Hkv, long rows) {
    const long R = (long)(Hq / Hkv) * Sq, pairs = (long)B * Hkv, cus = kv4_cus();
    auto plan = [&](int block, bool split) {
        Kv4TilePlan p;
        p.rows = block;
        p.blocks = (int)((R + block - 1) / block);
        const long most = (rows + 127) / 128, want = split ? 4 * cus / (pairs * p.blocks) : 1;
        p.ranges = (int)(want < 2 ? 1 : want > most ? most : want);
        return p;
    };
    // Up to 32 rows, drafts to be checked: four waves on one block of 32, which shares its tiles of 128 keys between them (32 x 5 tokens behind 4000 rows 59 us, as half of a block of
    // 64 73; 64 x 5 behind 1000 35 and 41; 8 x 6 behind 4000 29 and 31).  What is left of a tile's time is latency: one stage of LDS and two barriers a tile, two workgroups a CU.  Not where both the (sequence, kv head)s and their keys are few: a tile of 128 is a long wait then
    // (4 x 8 behind 500 18 us and, blocks of 64 in ranges, 15; 16 x 6 behind 800 24 and 23).
    if (R <= 32 && (pairs >= cus || rows >= 2048)) return plan(32, pairs < 2 * cus && rows >= 2048);
    // Blocks of 128 rows turn codes into operands for the most rows: where they fill the device (32 / 8 heads of 128, groups of 128, bf16: one prompt of 4096 rows 240 us, blocks
    // of 64 270; one of 2048 81 and 86), and, in ranges, where both rows and keys are many (512 tokens behind 3000 rows 67, blocks of 64 in ranges 74, whole 85).
    if (pairs * ((R + 127) / 128) >= 2 * cus) return plan(128, false);
    if (R >= 1024 && rows >= 2048) return plan(128, true);
    // Blocks of 64 leave two waves to a block of 32 rows, half of each tile's keys each, and a tile takes 1.6 us where it took 2.3: one prompt of 1200 rows 39 us, in blocks of
    // 128 48, those in ranges 58.  Ranges cost a launch more, 5 us and up: they pay for few blocks of 512 keys and more (4 x 40 tokens behind 2000 rows 33 us, whole 53; one prompt
    // of 300 rows 20, whole 16), of one for each CU only behind many keys (8 x 64 tokens behind 3000 rows 69, whole 77, behind 1000 38
    // and 33; 8 x 100 behind 2100, 448 blocks, 89 and 76).
    const long wgs = pairs * ((R + 63) / 64);
    return plan(64, wgs < cus ? rows >= 512 : 2 * wgs < 3 * cus && rows >= 2048);
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
    // (the smaller unit makes more workgroups: enough for either.  A cache of one unit is one workgroup's.)
    const long pairs = (long)B * num_kv_heads, rows = (long)pages_per_seq * page_rows;
    const int waves = kv4_waves(pairs, (long)R, rows);
    if (rows <= kv4_unit(1, waves)) return 0;
    return 2 * (size_t)kv4_stream_grid(pairs, kv4_unit(1, waves), waves, rows) * R * (head_dim + 4) * sizeof(float);
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
              out, Q, scale, is_causal, B, Sq, num_q_heads, nullptr, nullptr, nullptr, 0, 0, 0, nullptr};
    if (const int rc = paged_kv_check(who, a.c, page_rows, 4, group, head_dim)) return rc;
    MYNN_REQUIRE(dtype == MYNN_F16 || dtype == MYNN_BF16, MYNN_ERR_UNSUPPORTED, "%s: dtype %d: a 16-bit float type", who, dtype);
    a.c.page_shift = paged_shift(page_rows);
    MYNN_REQUIRE((long)num_q_heads * Sq < 1l << 30 && (long)B * num_kv_heads < 1l << 30, MYNN_ERR_UNSUPPORTED, "%s: B=%d Sq=%d heads %d", who, B, Sq, num_q_heads);
    const long rows = (long)pages_per_seq * page_rows;
    const size_t need = mynn_attention_paged_int4_workspace_bytes(B, Sq, pages_per_seq, page_rows, num_q_heads, num_kv_heads, head_dim);
    MYNN_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need), MYNN_ERR_INVALID, "%s: %zu bytes of workspace, %zu needed", who, workspace_bytes,
                 need);
    const size_t R = (size_t)(num_q_heads / num_kv_heads) * Sq;
    MYNN_REQUIRE((uintptr_t)counters % 4 == 0, MYNN_ERR_INVALID, "%s: unaligned counters", who);
    a.part_o = (float *)workspace;
    if (kv4_few_rows(num_q_heads, num_kv_heads, Sq)) {
        const long pairs = (long)B * num_kv_heads;
        const int fold = kv4_fold((long)R, head_dim / group), waves = kv4_waves(pairs, (long)R, rows), unit = kv4_unit(fold, waves);
        MYNN_REQUIRE(pairs * ((rows + unit - 1) / unit) < 1l << 30, MYNN_ERR_UNSUPPORTED, "%s: %d sequences of %d heads of %ld rows", who, B, num_kv_heads, rows);
        a.grid = kv4_stream_grid(pairs, unit, waves, rows);
        a.part_ml = a.part_o + 2 * (size_t)a.grid * R * head_dim;
        a.counters = counters;
        return dtype == MYNN_F16 ? kv4_stream_go<f16_t>(a, head_dim, group, fold, waves, as_stream(s)) : kv4_stream_go<bf16_t>(a, head_dim, group, fold, waves, as_stream(s));
    }
    const Kv4TilePlan plan = kv4_tile_plan(B, Sq, num_q_heads, num_kv_heads, rows);
    MYNN_REQUIRE((long)B * num_kv_heads * plan.blocks * plan.ranges < 1l << 24, MYNN_ERR_UNSUPPORTED, "%s: B=%d Sq=%d heads %d/%d", who, B, Sq, num_q_heads, num_kv_heads);
    a.grid = 2 * kv4_cus();
    a.blocks = plan.blocks;
    a.ranges = plan.ranges;
    const size_t lines = (size_t)plan.ranges * B * num_kv_heads * R;
    a.part_ml = a.part_o + lines * head_dim;
    a.length = (int *)(a.part_ml + lines * 2);
    return dtype == MYNN_F16 ? kv4_tile_go<f16_t>(a, head_dim, group, plan, as_stream(s)) : kv4_tile_go<bf16_t>(a, head_dim, group, plan, as_stream(s));
}
