// How large an entry point's operands may be and where they lie, so that it can refuse outputs that lie over what is read.
#pragma once

#include <initializer_list>
#include <stdint.h>

// The most rows, and values of one, that an entry point takes: its kernels count both in 32 bits and go past the last one, by a block's tiles or the
// pieces of its warps at most, before they ask.
constexpr int MOST = 0x7fffffff - 8192;

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
