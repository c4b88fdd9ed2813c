// Arithmetic on lengths and offsets that lie in device memory and that nobody
// has checked: whatever they hold, what comes out lies within what there is.
// Plain C++ (constexpr, so that device code may call it), compiled by a CPU test as well.
#pragma once

namespace ako_b200 {

constexpr int clamp_to(int x, int most) {
    const int y = x > 0 ? x : 0;
    return y < most ? y : most;
}

struct RowRange {
    int first, n;
};

// The rows begin .. end - 1 of `tokens`. Both ends are clamped before they are
// subtracted: begin and end may be any two numbers, and their difference none.
constexpr RowRange row_range(int begin, int end, int tokens) {
    const int first = clamp_to(begin, tokens), last = clamp_to(end, tokens);
    const int n = last - first;
    return {first, n > 0 ? n : 0};
}

// Position of new token `at` (0 <= at < n) of a sequence of kv_len tokens, the
// n new ones included, or -1 where the `held` positions of its table have no
// place for it. A length past the table moves no token onto an earlier one's place.
constexpr int new_position(int kv_len, int n, int at, int held) {
    const int p = (kv_len < 0 ? 0 : kv_len) - n + at;
    return p >= 0 && p < held ? p : -1;
}

}  // namespace ako_b200
