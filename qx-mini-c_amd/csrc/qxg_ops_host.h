// What the host sides of the operators on device memory (include/qxg.h) share: messages, and the checks of pointers,
// layouts and workspaces.  Header-only (internal linkage).
#pragma once
#include "qxg_ops.h"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cmath>

namespace {
struct Err {
    char *err;
    uint64_t n;
    __attribute__((format(printf, 2, 3))) bool operator()(const char *fmt, ...) const {
        if (err && n) {
            va_list ap;
            va_start(ap, fmt);
            vsnprintf(err, (size_t)n, fmt, ap);
            va_end(ap);
        }
        return false;
    }
};

// bytes of a value; 0 for another type
uint32_t type_size(uint32_t t) { return t == QXG_TYPE_F32 ? 4 : t == QXG_TYPE_F16 || t == QXG_TYPE_BF16 ? 2 : 0; }

struct Arg {
    const void *p;
    const char *name;
    bool need;         // may not be NULL
    uint32_t align;
};

// Runs `go` with the context's GPU current (and the caller's GPU again after it), once every pointer is
// known to be memory of that GPU.
template <size_t N, typename F>
bool on_device(const qxg_ctx *c, const Arg (&args)[N], hipStream_t s, int wait, const Err &fail, F go) {
    if (!c) return fail("invalid context");
    const int dev = qxg_ctx_device(c);
    // An error of this call is reported by it and cleared, unless the caller had one pending before.
    const bool pending = hipPeekAtLastError() != hipSuccess;
    const auto clear = [&] { if (!pending) (void)hipGetLastError(); };
    for (const Arg &a : args) {
        if (!a.p) continue;
        hipPointerAttribute_t at{};
        if (hipPointerGetAttributes(&at, a.p) != hipSuccess) {
            clear();
            return fail("%s is not device memory of this library's HIP runtime", a.name);
        }
        if (at.type != hipMemoryTypeDevice || at.device != dev) return fail("%s is not memory of the context's device %d", a.name, dev);
    }
    int before = dev;
    hipError_t e = hipGetDevice(&before);
    if (e == hipSuccess && before != dev) e = hipSetDevice(dev);
    if (e != hipSuccess) {
        clear();
        return fail("hipSetDevice failed");
    }
    e = go();
    if (wait) {   // also for what a launch that failed has left before it
        const hipError_t w = hipStreamSynchronize(s);
        if (e == hipSuccess) e = w;
    }
    if (before != dev) (void)hipSetDevice(before);
    if (e == hipSuccess) return true;
    clear();
    return fail("%s", hipGetErrorString(e));
}
template <size_t N> bool pointers_ok(const Arg (&args)[N], const Err &fail) {
    for (const Arg &a : args) {
        if (!a.p && a.need) return fail("%s is NULL", a.name);
        if ((uintptr_t)a.p % a.align) return fail("%s is not aligned to %u bytes", a.name, a.align);
    }
    return true;
}
// Whether rows of `row` elements at i a + j b, i < na, j < nb, overlap.  (Most layouts are nested: the rows of one
// index lie in a run of their own.)
bool rows_overlap(uint64_t a, uint64_t na, uint64_t b, uint64_t nb, uint64_t row) {
    using wide = unsigned __int128;
    if (na < nb) { std::swap(a, b); std::swap(na, nb); }
    if (na == 1) return false;
    if (a < row) return true;
    if (nb == 1) return false;
    if (b < row) return true;
    if (a >= (wide)(nb - 1) * b + row || b >= (wide)(na - 1) * a + row) return false;
    for (uint64_t j = 1; j < nb; ++j) {   // the two rows (i, 0) next to (0, j)
        const wide at = (wide)j * b, i = at / a;
        if ((i && i < na && at - i * a < row) || (i + 1 < na && (i + 1) * a - at < row)) return true;
    }
    return false;
}
// Rows of `row` bytes at p + i a + j b, i < na, j < nb
struct Rows {
    const void *p;
    const char *name;
    uint64_t a, na, b, nb, row;
};
// Whether rows of two arrays share memory.  Where the strides are the arrays' own, unlike ones, rows between each other's rows are not told
// apart: then it is whether the arrays' ranges meet.
bool rows_meet(const Rows &x, const Rows &y) {
    using wide = __int128;
    const auto size = [](const Rows &r) { return (wide)(r.na - 1) * r.a + (wide)(r.nb - 1) * r.b + r.row; };
    const wide d = (wide)(uintptr_t)y.p - (wide)(uintptr_t)x.p;
    if (d >= size(x) || -d >= size(y)) return false;
    if ((x.na > 1 && y.na > 1 && x.a != y.a) || (x.nb > 1 && y.nb > 1 && x.b != y.b)) return true;
    wide s = x.na > 1 ? x.a : y.a, t = x.nb > 1 ? x.b : y.b;
    // the rows' distances are d + i s + j t; they meet where one is between -y.row and x.row
    wide ilo = -(wide)(x.na - 1), ihi = y.na - 1, jlo = -(wide)(x.nb - 1), jhi = y.nb - 1;
    if (ihi - ilo > jhi - jlo) { std::swap(s, t); std::swap(ilo, jlo); std::swap(ihi, jhi); }
    const auto down = [](wide n, wide by) { return n / by - (n % by < 0); };
    for (wide i = ilo; i <= ihi; ++i) {
        const wide at = d + i * s, least = -(wide)y.row + 1 - at, most = (wide)x.row - 1 - at;   // of j t
        if (t == 0 ? least <= 0 && 0 <= most : std::max(jlo, -down(-least, t)) <= std::min(jhi, down(most, t))) return true;
    }
    return false;
}
uint64_t up16(uint64_t v) { return (v + 15) & ~15ull; }
bool workspace_ok(const void *p, uint64_t have, uint64_t need, const Err &fail) {
    return !need || (p && have >= need) || fail("the workspace holds %llu bytes; this call needs %llu", (unsigned long long)(p ? have : 0), (unsigned long long)need);
}
}  // namespace
