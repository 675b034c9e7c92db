// Where the pieces of a (row, head) pair's sums lie in the workspace of the attention over the 4-bit cache
// (csrc/kv4_attn.hip). Plain C++ (no HIP), so that a test walks it on the host.
//
// split4_kernel has places 0 .. split - 1, kRows for each of its workgroups. Behind them, where a call may have row tiles
// (`all` > `split`), lie two regions of kPromptFill x kPromptRows places for prompt4_kernel's workgroups.
#pragma once

namespace qk {

constexpr int kRows = 8;               // (row, head) pairs of a split4_kernel workgroup
constexpr int kPromptRows = 128;       // and of a prompt4_kernel workgroup
constexpr int kPromptFill = 256;       // prompt4_kernel's workgroups of a call whose units are cut
constexpr int kPromptRegion = kPromptFill * kPromptRows;

// Where the pieces of a unit lie. split4_kernel's are neighbours, kRows places each. A workgroup of prompt4_kernel has kPromptRows
// places for the piece that ends its first unit, or passes through it, and in a second region as many for the one that begins its
// last.
struct Places {
    int first, rows, second;   // of a row: the first piece's place in the first region; the second region's distance, or 0
    constexpr int of(int piece) const { return first + (piece == 0 ? second : piece * rows); }
};
constexpr Places places_of(int first, int split) {
    return first < split ? Places{first, kRows, 0} : Places{first, kPromptRows, kPromptRegion};
}

// Whether `pieces` pieces from `first` on are there to be joined: more than one, each at a place of the workspace. (One piece is
// in the output already, and where starts decrease an entry may be anything that the workspace held.)
constexpr bool joinable(int first, int pieces, int split, int all) {
    if (first < 0 || pieces < 2) return false;
    const Places p = places_of(first, split);
    const int end = p.second ? all - p.second : split;   // of the region that the pieces but the first are in
    return first < end && pieces <= (end - first - 1) / p.rows + 1;
}

}  // namespace qk
