// Rows of heads in memory: whether an output lies over an input.  Host code, without HIP.
#pragma once

#include "../../include/spy_hip.h"

// Whether two tensors of the same rows share memory, as far as their strides say so: one lies over the first or last piece (a row's head) of the other and leaves no gap there,
// or both are parts of wider rows and a head of one meets a head of the other.  Rows that are told apart in no such way are the caller's to keep apart.
static inline bool pg_rows_meet(const spy_hip_tensor *a, const spy_hip_tensor *b) {
    struct rows { uintptr_t at; int64_t w, h, r, nh, nr, size; bool dense; };
    const auto of = [](const spy_hip_tensor *t) {
        rows x = {(uintptr_t)t->data, t->ne[0] * t->nb[0], t->nb[1], t->nb[2], t->ne[1], t->ne[2], 0, false};
        x.size = (x.nh - 1) * x.h + (x.nr - 1) * x.r + x.w;
        x.dense = x.size == x.w * x.nh * x.nr;
        return x;
    };
    const rows x = of(a), y = of(b);
    if (x.at + x.size <= y.at || y.at + y.size <= x.at) return false;
    if (x.at == y.at) return true;
    const auto covers = [](const rows &p, const rows &q) {
        const uintptr_t last = q.at + q.size - q.w;
        return p.dense && ((q.at < p.at + p.size && q.at + q.w > p.at) || (last < p.at + p.size && last + q.w > p.at));
    };
    if (covers(x, y) || covers(y, x)) return true;
    if (x.r != y.r || (x.nh - 1) * x.h + x.w > x.r || (y.nh - 1) * y.h + y.w > y.r) return false;
    // y's heads from x's on, by rows of x: in row `shift` from `in` on, and, where a head reaches past that row's end, in the next one
    const int64_t off = (int64_t)(y.at - x.at), shift = off >= 0 ? off / x.r : -((-off + x.r - 1) / x.r), in = off - shift * x.r;
    const auto meets = [&](int64_t from) {                                 // a head of y's row, `from` bytes into a row of x, and one of x's
        for (int64_t i = 0, j = 0; i < x.nh && j < y.nh;) {
            const int64_t p = i * x.h, q = from + j * y.h;
            if (p + x.w <= q) i++;
            else if (q + y.w <= p) j++;
            else return true;
        }
        return false;
    };
    return (shift < x.nr && -shift < y.nr && meets(in)) || (shift + 1 < x.nr && -shift - 1 < y.nr && meets(in - x.r));
}
