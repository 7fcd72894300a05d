// stratametal_amd/csrc/smoe_check.hpp - argument checks of the C ABI's operators (smoe_dense.cpp, smoe_attention.cpp): the
// thread's last error, alignments, and which bytes two buffers share.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "smoe.h"

namespace smoe {

smoe_status report(smoe_status s, const std::string& why);  // smoe_api.cpp: the thread's last error

inline smoe_status fail(smoe_status s, const std::string& why) { return report(s, why); }
inline smoe_status ok() { return report(SMOE_OK, ""); }
inline smoe_status launched(hipError_t e, const char* what) {
    return e == hipSuccess ? ok() : fail(SMOE_EDEVICE, std::string(what) + ": " + hipGetErrorString(e));
}

inline bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
inline bool elem_type(int32_t t) { return t == SMOE_F32 || t == SMOE_F16 || t == SMOE_BF16; }
inline size_t elem_size(int32_t t) { return t == SMOE_F32 ? 4 : 2; }
inline bool finite(float v) { return std::isfinite(v); }

// `rows` rows of `width` bytes, `step` bytes apart.
struct Span {
    const void* p;
    int64_t rows, step, width;
    uintptr_t lo() const { return (uintptr_t)p; }
    uintptr_t hi() const { return lo() + (uintptr_t)((rows - 1) * step + width); }
};
inline Span rows_of(const void* p, int32_t type, int64_t rows, int64_t ld, int64_t n) {
    const int64_t es = (int64_t)elem_size(type);
    return {p, rows, rows > 1 ? ld * es : n * es, n * es};
}
inline Span bytes_of(const void* p, int64_t bytes) { return {p, 1, bytes, bytes}; }
// Whether a written span shares a byte with another: columns of one matrix (the same step) that lie apart do not, nor does
// one row between the rows of a matrix.
inline bool overlap(const Span& a, const Span& b) {
    if (!a.p || !b.p || a.hi() <= b.lo() || b.hi() <= a.lo()) return false;
    if (a.rows == 1 && b.rows > 1) return overlap(b, a);
    if (b.rows == 1 && a.step >= a.width) {
        const int64_t from = (int64_t)(b.lo() - a.lo());  // of a's rows, the first that ends past b's start
        const int64_t i = from < a.width ? 0 : (from - a.width) / a.step + 1;
        return i < a.rows && i * a.step < from + b.width;
    }
    if (a.step != b.step || a.step < a.width || a.step < b.width) return true;
    const int64_t at = ((int64_t)(b.lo() - a.lo()) % a.step + a.step) % a.step;  // b's rows within a's step
    return at < a.width || at + b.width > a.step;
}
// The same rows: an element is read by the thread that then writes it.
inline bool same(const Span& a, const Span& b) { return a.p == b.p && a.step == b.step && a.width == b.width; }

// Row strides of 2^40 values and more cannot be those of memory (and would overflow the byte offsets).
constexpr int64_t kMaxLd = (int64_t)1 << 40;
inline bool bad_ld(int64_t ld, int64_t rows, int64_t least) { return rows > 1 && (ld < least || ld > kMaxLd); }

}  // namespace smoe
