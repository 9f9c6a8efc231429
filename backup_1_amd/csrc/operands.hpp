// Where the operands of a call lie to each other, on the host: whether a result meets an input or another result.
#pragma once
#include <cstddef>
#include <cstdint>
#include <initializer_list>

namespace decx_hip {

// `rows` rows of `width` bytes, `pitch` bytes apart (pitch >= width); p = nullptr: not there
struct Operand {
    const void* p = nullptr;
    size_t rows = 0, width = 0, pitch = 0;
    uintptr_t begin() const { return reinterpret_cast<uintptr_t>(p); }
    uintptr_t end() const { return begin() + (rows - 1) * pitch + width; }
    bool there() const { return p && rows && width; }
};
inline Operand operand(const void* p, size_t rows, size_t cols, size_t ld, size_t size) { return {p, rows, cols * size, ld * size}; }

// Whether they have a byte in common.  Rows of two operands may lie between each other (columns of one matrix): equal pitches are
// compared as such, rows of unequal ones one by one, which takes time only where operands that wide apart are nested.
inline bool operands_meet(const Operand& a, const Operand& b) {
    if (!a.there() || !b.there() || a.end() <= b.begin() || b.end() <= a.begin()) return false;
    const Operand &few = a.rows <= b.rows ? a : b, &many = a.rows <= b.rows ? b : a;
    // the rows of `many` that bytes from..to meet begin before `to` and end after `from`
    auto row_meets = [&](uintptr_t from, uintptr_t to) {
        if (to <= many.begin() || from >= many.end()) return false;
        const size_t first = from < many.begin() + many.width ? 0 : (from - many.begin() - many.width) / many.pitch + 1;
        return first < many.rows && many.begin() + first * many.pitch < to;
    };
    if (few.pitch != many.pitch || few.rows == 1) {
        for (size_t i = 0; i < few.rows; ++i)
            if (row_meets(few.begin() + i * few.pitch, few.begin() + i * few.pitch + few.width)) return true;
        return false;
    }
    // one pitch: row i of `few` lies at the same place between two rows of `many` for every i, so the first row of it that is not
    // before `many`, the one before that and the last decide
    const size_t at = few.begin() < many.begin() ? (many.begin() - few.begin()) / few.pitch : 0;
    for (size_t i = at; i < few.rows && i <= at + 1; ++i)
        if (row_meets(few.begin() + i * few.pitch, few.begin() + i * few.pitch + few.width)) return true;
    return false;
}
inline bool operands_coincide(const Operand& a, const Operand& b) {
    return a.p == b.p && a.rows == b.rows && a.width == b.width && (a.rows == 1 || a.pitch == b.pitch);
}

// A result, and which inputs (bit i: number i of the call's list) it may lie exactly over
struct Result {
    Operand at;
    unsigned over = 0;
};
// The results meet no input but one that they may lie over and then coincide with, and none of each other
inline bool results_fit(std::initializer_list<Result> results, std::initializer_list<Operand> inputs) {
    for (const Result* r = results.begin(); r != results.end(); ++r) {
        unsigned bit = 1;
        for (const Operand& in : inputs) {
            if (operands_meet(r->at, in) && !((r->over & bit) && operands_coincide(r->at, in))) return false;
            bit <<= 1;
        }
        for (const Result* o = r + 1; o != results.end(); ++o)
            if (operands_meet(r->at, o->at)) return false;
    }
    return true;
}

}  // namespace decx_hip
