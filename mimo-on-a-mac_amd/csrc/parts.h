// Where the parts of a split row tile begin.  Plain C++, so that the host can check it at lengths that no test's cache holds.
#pragma once

namespace mimo {

// floor(i units / parts), 0 <= i <= parts <= 2^15: part i is units part_begin(i) .. part_begin(i + 1) - 1.  The product itself
// passes 32 bits (512 parts of 2^22 units, 2^28 keys), so the quotient of units by parts is multiplied apart from its rest.
constexpr int part_begin(int i, int units, int parts) { return i * (units / parts) + i * (units % parts) / parts; }

}  // namespace mimo
