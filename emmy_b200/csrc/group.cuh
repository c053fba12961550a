// Rows grouped by a key on the device: the blocks of rows of one adapter (lora.cu) or of one expert (moe_w8.cu).
#pragma once
#include "common.cuh"

namespace eq {

struct GroupBlock {
    int32_t key;    // -1: rows whose id is no key
    int32_t first;  // in the list of rows
    int32_t count;  // 1 to block_rows
    int32_t note;   // not written here: the caller's own
};

// Most blocks that T rows of `keys` keys can make (rows whose id is no key count as one more).
inline int64_t group_max_blocks(int64_t T, int64_t keys, int64_t block_rows, bool cut) {
    const int64_t kinds = keys + 1 < T ? keys + 1 : T;  // every kind has at most one block that is not full, two where it is cut
    const int64_t most = (cut ? 2 : 1) * kinds + T / block_rows;
    return most < T ? most : T;
}

// rows[0, ..): the indices 0 .. T - 1 in order of their ids (those outside [0, keys) last, or left out unless keep_rest); blocks: each at
// most block_rows (a power of two) rows of one key; n_blocks: how many; status (may be null): set to zero.  The rows of a key stay in their order.  One launch, a
// programmatic dependent.  cut: a key's rows are cut ahead of the last run of neighbours among them (kGroupRun rows and more), so that the prompt behind a few
// rows that decode lies in blocks of neighbours.
constexpr int kGroupMaxKeys = 4096;
constexpr int kGroupRun = 32;
int group_rows_launch(const int32_t* ids, int T, int keys, bool keep_rest, int block_rows, bool cut, GroupBlock* blocks, int32_t* n_blocks, int32_t* rows,
                      int* status, cudaStream_t stream);

}  // namespace eq
