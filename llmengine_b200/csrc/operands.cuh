// Where an entry point's operands lie, so that it can refuse outputs that lie over what is read.
#pragma once

#include <initializer_list>
#include <stdint.h>

struct Span { uintptr_t first, end, width, pitch; };       // bytes: from, to, of a row, from row to row; empty where there is no operand

// rows x cols values of `bytes` each, `stride` values from row to row
inline Span span(const void* at, long long rows, long long cols, long long stride, int bytes) {
    if (!at || rows <= 0 || cols <= 0) return {0, 0, 0, 0};
    const uintptr_t first = (uintptr_t)at, width = (uintptr_t)(cols * bytes), pitch = (uintptr_t)(stride * bytes);
    return {first, first + (uintptr_t)(rows - 1) * pitch + width, width, pitch};
}
// Whether two operands share a byte.  Rows of one pitch may stand side by side in one buffer; of other pitches only what lies apart is apart.
inline bool meets(const Span& a, const Span& b) {
    if (a.first >= b.end || b.first >= a.end) return false;
    if (a.pitch != b.pitch || a.pitch == 0) return true;
    const uintptr_t apart = b.first >= a.first ? (b.first - a.first) % a.pitch : (a.pitch - (a.first - b.first) % a.pitch) % a.pitch;
    return apart < a.width || apart + b.width > a.pitch;
}
inline bool meets(const Span& out, std::initializer_list<Span> others) {
    for (const Span& o : others)
        if (meets(out, o)) return true;
    return false;
}
