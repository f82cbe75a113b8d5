// Trees of drafted tokens over a cache in pages: the kernel of attention_prompt.h, with rows that see the whole context and, of
// their own tree, what their masks say.  A row's place among the keys plays no part but in a window, which is held against the
// depth in the tree.
//
// Between a token and a prompt: n rows of a group of G query heads make 4 * head_dim * n * G operations for 4 * head_dim bytes of a key
// and value, so small trees are bound by HBM and trees past some 190 / G rows by the matrix cores.  There are few tiles (a tree of 32 rows under a
// group of four is one) over contexts of any length, so the keys of all tiles are cut into parts that fill the card once; the
// lengths are on the device only, and every workgroup finds its part from them (tree_work).
//
// Measured on one MI355X: 4 trees of 64 over 32768 under 64 heads on 8 306 us, 0.9 PFLOP/s (the matrix cores: what a library's large
// product reaches would be 200 us); 24 trees up to 16 over contexts up to 8191 under 32 heads on 8 37 us, 3.1 TB/s; 32 trees
// up to 12 on an int8 cache under a window of 4096 37 us; two trees of 117 over 6001 under 14 heads on 2 32 us; 7 drafted tokens
// over 997 15 us.  The last three are chains of waits: finding the part 1.5 to 3 us, pages, addresses and the first rows 3, some
// 1.1 us a step of 64 keys, the joins.
#include "attention_prompt.h"

namespace qk {

void launch_attention_few_rows(const void* args, int64_t grid, hipStream_t stream);

namespace {

// Rows of a tree and key-value head, on average, up to which tiles are of 64 rows (32 trees of up to 48 rows on an int8 cache 37 us, in
// tiles of 128 53; 16 trees over 4096 of 48 rows 64.5 and 67.6, of 64 65.2 and 68.5, of 96 74.5 and 72.9, of 192 112 and 90).
constexpr int64_t kFewRows = 64;

struct Plan {
    int64_t grid, arrivals_bytes, part_bytes, parts, tiles;
    int room;
    bool half;
};

Plan plan(int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache& c, int64_t table_width) {
    Plan p = {};
    const int64_t some = batch < tokens ? batch : tokens;
    // at most, of a key-value head: row tiles, and parts of a tile
    const int64_t group = q_heads / c.kv_heads;
    p.half = tokens * group <= kFewRows * batch;
    const int64_t rows = p.half ? kRows / 2 : kRows;
    const int64_t tiles = p.tiles = tokens * group / rows + some + 1;
    const int64_t parts = table_width * c.page_size / kKeys / kTreeSteps + 1;
    // cut tiles fill the card's places once; heads wider than 128 leave one workgroup per CU
    const int64_t room = (c.head_dim <= 128 ? kResident : kResident / 2) / c.kv_heads;
    p.room = room < 1 ? 1 : (int)room;
    // How many tiles there are is known on the device only: tiles that are not cut, or parts that fill the room.  Workgroups without
    // a part end at once.
    const int64_t ranks = tiles > p.room ? tiles : tiles * parts < p.room ? tiles * parts : p.room;
    p.grid = ranks * c.kv_heads;
    if (p.room > 1 && parts > 1) {
        p.parts = (ranks < p.room ? ranks : p.room) * c.kv_heads;
        p.arrivals_bytes = ((tiles * c.kv_heads + p.parts) * 8 + 255) / 256 * 256;
        p.part_bytes = rows * (padded_width(c) + 2) * 4;
    }
    return p;
}

}  // namespace

size_t attention_tree_workspace(int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache& c, int64_t table_width) {
    if (tokens == 0) return 0;
    const Plan p = plan(tokens, batch, q_heads, c, table_width);
    return (size_t)(p.arrivals_bytes + p.parts * p.part_bytes);
}

hipError_t launch_attention_tree(const AttnArgs& a, const TreeMask& mask, void* workspace, hipStream_t stream) {
    const Plan p = plan(a.tokens, a.batch, a.q_heads, a.kv.c, a.kv.table_width);
    PromptArgs g = {};
    g.a = a;
    g.group_div = div31((uint32_t)(a.q_heads / a.kv.c.kv_heads));
    g.splits = p.room;
    g.mask = mask;
    g.most_tiles = p.tiles;
    if (p.parts > 0) {
        g.tag = next_split_tag();
        g.arrivals = (uint64_t*)workspace;
        g.group_arrivals = g.arrivals + p.tiles * a.kv.c.kv_heads;
        g.parts = (float*)((char*)workspace + p.arrivals_bytes);
        g.part_bytes = p.part_bytes;
    }
    if (p.half) launch_attention_few_rows(&g, p.grid, stream);
    else launch_form<true>(g, p.grid, stream);
    return hipGetLastError();
}

}  // namespace qk
