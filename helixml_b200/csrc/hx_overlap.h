// Whether two strided operands share memory: what entry points refuse whose kernels read an operand after they began to write another.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace hx {

// outer x inner rows of `bytes` bytes each; strides in bytes, >= 0.
struct Rows {
    const void *at;
    int64_t outer, outer_stride, inner, inner_stride, bytes;
};
inline Rows rows_of(const void *at, int64_t batch, int64_t batch_stride, int64_t rows, int64_t row_stride, int64_t columns, size_t element) {
    const int64_t e = (int64_t)element;
    return {at, batch, batch_stride * e, rows, row_stride * e, columns * e};
}
inline Rows dense_of(const void *at, int64_t bytes) { return {at, 1, 0, 1, 0, bytes}; }

namespace overlap_detail {
inline int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b != 0 && a < 0); }   // b > 0
// Whether lo < k * s < hi for an integer k in k0 .. k1.
inline bool multiple_between(int64_t lo, int64_t hi, int64_t s, int64_t k0, int64_t k1) {
    if (s == 0) return lo < 0 && 0 < hi && k0 <= k1;
    return std::max(k0, floor_div(lo, s) + 1) <= std::min(k1, floor_div(hi - 1, s));
}
}  // namespace overlap_detail

// Some byte of a is a byte of b.  Exact: halves of one buffer do not overlap, although their extents do.  A row of a and a row of b are
// delta + i S + j s apart; where both have the same strides, i and j run over the differences of their indices and a handful of i can
// matter.  Otherwise the rows of b are held against a one by one, which no ordinary pair of operands comes to.
inline bool overlap(Rows a, Rows b) {
    using namespace overlap_detail;
    for (Rows *r : {&a, &b}) {
        if (r->at == nullptr || r->outer <= 0 || r->inner <= 0 || r->bytes <= 0) return false;
        if (r->outer_stride == 0) r->outer = 1;
        if (r->inner_stride == 0) r->inner = 1;
        if (r->outer == 1) r->outer_stride = 0;
        if (r->inner == 1) r->inner_stride = 0;
    }
    auto extent = [](const Rows &r) { return (r.outer - 1) * r.outer_stride + (r.inner - 1) * r.inner_stride + r.bytes; };
    const int64_t delta = (int64_t)((uintptr_t)b.at - (uintptr_t)a.at);   // b's first row from a's
    if (delta >= extent(a) || -delta >= extent(b)) return false;
    auto alike = [](int64_t s, int64_t n, int64_t t, int64_t m) { return s == t || n == 1 || m == 1; };
    if (alike(a.outer_stride, a.outer, b.outer_stride, b.outer) && alike(a.inner_stride, a.inner, b.inner_stride, b.inner)) {
        int64_t S = std::max(a.outer_stride, b.outer_stride), s = std::max(a.inner_stride, b.inner_stride);
        int64_t i0 = 1 - a.outer, i1 = b.outer - 1, j0 = 1 - a.inner, j1 = b.inner - 1;
        if (S < s) std::swap(S, s), std::swap(i0, j0), std::swap(i1, j1);
        // -b.bytes < delta + i S + j s < a.bytes
        const int64_t lo = -b.bytes - delta, hi = a.bytes - delta;
        if (S > 0) {
            i0 = std::max(i0, floor_div(lo - j1 * s, S) + 1);
            i1 = std::min(i1, floor_div(hi - 1 - j0 * s, S));
        }
        for (int64_t i = i0; i <= i1; ++i)
            if (multiple_between(lo - i * S, hi - i * S, s, j0, j1)) return true;
        return false;
    }
    if (a.outer_stride < a.inner_stride) std::swap(a.outer, a.inner), std::swap(a.outer_stride, a.inner_stride);
    const int64_t block = (a.inner - 1) * a.inner_stride + a.bytes;   // of a's outer index
    for (int64_t i = 0; i < b.outer; ++i)
        for (int64_t j = 0; j < b.inner; ++j) {
            const int64_t q = delta + i * b.outer_stride + j * b.inner_stride;   // this row of b from a's first
            int64_t k0 = 0, k1 = a.outer - 1;
            if (a.outer_stride > 0) {
                k0 = std::max<int64_t>(k0, floor_div(q - block, a.outer_stride) + 1);
                k1 = std::min<int64_t>(k1, floor_div(q + b.bytes - 1, a.outer_stride));
            }
            for (int64_t k = k0; k <= k1; ++k)
                if (multiple_between(q - k * a.outer_stride - a.bytes, q - k * a.outer_stride + b.bytes, a.inner_stride, 0, a.inner - 1)) return true;
        }
    return false;
}

// An operand of a call, for the message that refuses it.
struct Operand {
    const char *name;
    Rows rows;
};
// The first of `outs` that shares memory with one of `ins` or another of `outs`, and that other one; or false.
template <size_t N, size_t M>
inline bool shared_operands(const Operand (&outs)[N], const Operand (&ins)[M], const char *&first, const char *&second) {
    for (size_t i = 0; i < N; ++i)
        for (size_t j = i + 1; j < N + M; ++j) {
            const Operand &other = j < N ? outs[j] : ins[j - N];
            if (overlap(outs[i].rows, other.rows)) {
                first = outs[i].name, second = other.name;
                return true;
            }
        }
    return false;
}

}  // namespace hx
