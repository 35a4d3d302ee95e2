// Checks of strided tensors of heads, of small arrays and of scratch, shared by the
// entry points for tokens.
#pragma once

#include <string>

#include "capi_context.hpp"

namespace mh {
namespace capi {

inline size_t size_of(WeightType t) { return t == kF16 ? 2 : 4; }

// A strided tensor of heads: its rows' elements and where they lie.
struct Rows {
    const char *p;
    int64_t rows, ld, cols;
    size_t size;
    const char *end() const { return p + (rows ? size_t((rows - 1) * ld + cols) * size : 0); }
};

inline Rows rows_of(const void *p, uint64_t rows, uint32_t heads, uint32_t d, uint64_t ld, WeightType t,
             const char *what) {
    const std::string name = what;
    if (heads == 0 || d == 0) fail(kInvalidArgument, name + ": no heads or channels");
    const uint64_t cols = uint64_t(dim(heads, "heads")) * uint64_t(dim(d, "d"));
    if (cols > (1u << 30)) fail(kInvalidArgument, name + ": row too large");
    if (ld < cols) fail(kInvalidArgument, name + ": ld is less than heads * d");
    if (ld > (uint64_t(1) << 40) || (rows && ld > (uint64_t(1) << 60) / rows))
        fail(kInvalidArgument, name + ": tensor too large");
    if (rows) need(p, what);
    if (reinterpret_cast<uintptr_t>(p) % size_of(t)) fail(kInvalidArgument, name + " is not aligned to its type");
    return Rows{static_cast<const char *>(p), int64_t(rows), int64_t(ld), int64_t(cols), size_of(t)};
}

// Whether a and b share elements: ranges that meet, unless their rows step alike and
// their columns lie apart.
inline bool overlap(const Rows &a, const Rows &b) {
    if (!a.rows || !b.rows || a.p >= b.end() || b.p >= a.end()) return false;
    if (a.ld != b.ld || a.size != b.size) return true;
    const int64_t step = a.ld * int64_t(a.size);
    int64_t off = (b.p - a.p) % step;
    if (off < 0) off += step;
    return off < a.cols * int64_t(a.size) || off + b.cols * int64_t(b.size) > step;
}

inline void no_overlap(const Rows &a, const Rows &b, const char *what) {
    if (overlap(a, b)) fail(kInvalidArgument, std::string(what) + " overlap");
}

// The same place (in place), or apart.
inline void same_or_apart(const Rows &in, const Rows &out, const char *what) {
    if (in.p == out.p && in.ld == out.ld) return;
    no_overlap(in, out, what);
}

// Arrays of 4-byte elements (NULL counts as aligned).
inline void aligned4(const void *p, const char *what) {
    if (reinterpret_cast<uintptr_t>(p) % 4)
        fail(kInvalidArgument, std::string(what) + " is not aligned to its type");
}

// The caller's scratch, or NULL where the context's workspace is to be used.
inline void *check_scratch(Context &c, void *scratch, uint64_t bytes, size_t needed) {
    if (!needed) return nullptr;
    if (scratch) {
        if (bytes < needed) fail(kInvalidArgument, "scratch is smaller than this call needs");
        if (!aligned16(scratch)) fail(kInvalidArgument, "scratch is not 16-byte aligned");
        return scratch;
    }
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    HIP_CHECK(hipStreamIsCapturing(c.stream, &st));
    if (st != hipStreamCaptureStatusNone)
        fail(kInvalidArgument, "a captured call needs scratch of its own: the context's workspace may move");
    return nullptr;
}

}  // namespace capi
}  // namespace mh
