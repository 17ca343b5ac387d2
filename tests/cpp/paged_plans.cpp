// The rules by which the paged attention and the log probabilities are launched
// (csrc/paged_plan.hpp, logprobs_plan.hpp) behind C functions, for the CPU tests.
#include "../../atlas_amd/csrc/logprobs_plan.hpp"
#include "../../atlas_amd/csrc/paged_plan.hpp"

extern "C" {

// out: units of a whole row (0: rows are split), wavefronts, few_parts, most_parts, lanes, threads and workgroups of the join
void attention_plan(int format, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim, uint32_t sequences, uint32_t table_width,
                    uint32_t q_heads, uint32_t window, uint32_t* out) {
    const atlas::PagedCache c{nullptr, nullptr, 1, page_size, kv_heads, head_dim, sequences, table_width, format};
    const atlas::PagedPlan p = atlas::paged_plan(c, q_heads);
    const uint64_t rows = atlas::paged_rows(c, q_heads);
    out[0] = atlas::whole_row_units(c, window, rows);
    out[1] = out[0] ? atlas::paged_waves(format, (head_dim + 31) / 32, out[0], rows) : atlas::kPagedAttnWaves;
    out[2] = p.few_parts;
    out[3] = p.most_parts;
    const atlas::PagedJoin j = atlas::paged_join(c, q_heads, p.most_parts);
    out[4] = j.lanes;
    out[5] = j.threads;
    out[6] = j.groups;
}

// out: strips of a row, strips of a slice, slices of a row, workgroups of the first launch, threads of the second's
void logprobs_plan(uint32_t rows, uint32_t vocab, uint32_t* out) {
    out[0] = atlas::strips_of(vocab);
    out[1] = atlas::strips_each(rows, vocab);
    out[2] = atlas::slices_of(rows, vocab);
    out[3] = atlas::sum_groups(rows, vocab);
    out[4] = atlas::row_threads(rows);
}
}
