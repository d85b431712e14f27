// How few long rows of class logits are cut over workgroups (label_dist.hip, sampling).  Plain C++: its arithmetic, up to 2^31 - 1 classes, is
// checked on the host.
#pragma once
#include <algorithm>

namespace mh {
namespace ld {

struct RowCut {
    int nseg, length;           // workgroups a row (0: not cut), classes of each but the last
};
// Where the rows alone do not fill half of the chip, as many workgroups as fill it, of at least 4096 classes, a multiple of 8
inline RowCut row_cut(int rows, int classes)
{
    if (rows <= 0 || rows > 128 || classes < 16384) return RowCut{0, 0};
    const int want = std::max(2, std::min(256 / rows, classes / 4096));
    const long long n = classes, length = ((n + want - 1) / want + 7) / 8 * 8;
    return RowCut{(int)((n + length - 1) / length), (int)length};
}

}  // namespace ld
}  // namespace mh
