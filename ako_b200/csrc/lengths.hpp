// Arithmetic on lengths and offsets that lie in device memory and that nobody
// has checked: whatever they hold, what comes out lies within what there is.
// Plain C++ (constexpr, so that device code may call it), compiled by a CPU test as well.
#pragma once

namespace ako_b200 {

constexpr int clamp_to(int x, int most) { return x < 0 ? 0 : x < most ? x : most; }

struct RowRange {
    int first, n;
};

// The rows begin .. end - 1 of `tokens`. Both ends are clamped before they are
// subtracted: begin and end may be any two numbers, and their difference none.
constexpr RowRange row_range(int begin, int end, int tokens) {
    const int first = clamp_to(begin, tokens), last = clamp_to(end, tokens);
    return {first, last > first ? last - first : 0};
}

}  // namespace ako_b200
