// fattn_pieces.h -- how many pieces the open tiles of a query block are cut into
// by the scored attention of many queries (k_fattn_scored.hip). Plain C++, which
// the kernel's workgroups evaluate each for itself.
#pragma once

namespace mi355x {

constexpr int kFsLengths = 512;  // lengths that a launch looks at, a thread each

// n open tiles in pieces of at most len, but no more than most
constexpr int fs_pieces(int n, int len, int most) {
    const int p = (int) ((float) (n + len - 1) / (float) len), q = p < most ? p : most;
    return q > 1 ? q : 1;
}

// The i-th length: from four tiles on in equal steps. The last is a whole span's at
// least, a piece a block, which has a place on the card wherever blocks are cut at all
constexpr int fs_length(int i, int n_tiles) {
    const int step = (n_tiles - 4 + kFsLengths - 2) / (kFsLengths - 1);
    return 4 + i * (step > 1 ? step : 1);
}

}  // namespace mi355x
