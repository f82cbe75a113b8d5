// Prompts: how the kernel of attention_prompt.h is launched for them.
#include "attention_prompt.h"

namespace qk {
namespace {

struct Plan {
    int64_t grid, arrivals_bytes, part_bytes;
    int splits;
};

Plan plan(int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache& c, int64_t table_width, int64_t window, int64_t sinks) {
    Plan p = {};
    const int64_t group = q_heads / c.kv_heads;
    // at most: whole tiles, and a last one for every sequence and for the rows past them
    const int64_t some = batch < tokens ? batch : tokens;
    const int64_t tiles = (tokens * group / kRows + some + 1) * c.kv_heads;
    int64_t most = (table_width ? table_width : 1) * c.page_size;
    if (window && most > window && most - window > sinks + kRows) most = window + sinks + kRows;
    const int64_t steps = (most + kKeys - 1) / kKeys;
    int64_t splits = kResident / tiles;
    if (splits > steps / kSplitTiles) splits = steps / kSplitTiles;
    p.splits = splits < 1 ? 1 : (int)splits;
    p.grid = tiles * p.splits;
    if (p.splits > 1) {
        p.arrivals_bytes = (tiles * 8 + 255) / 256 * 256;
        p.part_bytes = kRows * (padded_width(c) + 2) * 4;
    }
    return p;
}

}  // namespace

size_t attention_prompt_workspace(int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache& c, int64_t table_width,
                                  int64_t window, int64_t sinks) {
    if (tokens == 0) return 0;
    const Plan p = plan(tokens, batch, q_heads, c, table_width, window, sinks);
    return (size_t)(p.arrivals_bytes + p.grid * p.part_bytes);
}

hipError_t launch_attention_prompt(const AttnArgs& a, void* workspace, hipStream_t stream) {
    const Plan p = plan(a.tokens, a.batch, a.q_heads, a.kv.c, a.kv.table_width, a.window, a.sinks);
    PromptArgs g = {};
    g.a = a;
    g.group_div = div31((uint32_t)(a.q_heads / a.kv.c.kv_heads));
    g.splits = p.splits;
    if (p.splits > 1) {
        g.tag = next_split_tag();
        g.arrivals = (uint64_t*)workspace;
        g.parts = (float*)((char*)workspace + p.arrivals_bytes);
        g.part_bytes = p.part_bytes;
    }
    launch_form<false>(g, p.grid, stream);
    return hipGetLastError();
}

}  // namespace qk
