// Trees of few rows: the kernel of attention_prompt.h with tiles of 64 rows, in a file of its own so that it is compiled beside the
// others.
//
// With 64 rows a tile of 128 would leave two of the four waves without any, and one step after another of the other two would take
// longer than its keys take to come.  Here two waves take the first 32 keys of every step, two the others, half as long each; their
// sums are joined once, at the end of a workgroup's part.
#include "attention_prompt.h"

namespace qk {

void launch_attention_few_rows(const void* args, int64_t grid, hipStream_t stream) {
    launch_form<true, true>(*(const PromptArgs*)args, grid, stream);
}

}  // namespace qk
