// Host-side helpers of the libqim C ABI: error reporting and argument checks.
#pragma once

#include <atomic>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <tuple>
#include <type_traits>
#include <utility>

#include "qim.h"

namespace qim {

// Records a message for qim_last_error() and returns `code`.
int fail(int code, const char *fmt, ...);

// First failed launch of the current entry point on this host thread
// (hipSuccess if none); launch() sets it, check_launch() reads and resets it.
hipError_t &launch_error();

// kernel<<<grid, block, shmem, stream>>>(args...) through hipLaunchKernel,
// whose return value is the status of this launch alone.  (hipGetLastError
// after a triple-chevron launch would also report an earlier failure of any
// runtime call on this thread, torch's included, as this launch's.)
template <typename... P, size_t... I>
hipError_t launch_packed(const void *fn, dim3 grid, dim3 block, size_t shmem, hipStream_t stream,
                         std::tuple<P...> &vals, std::index_sequence<I...>) {
    void *ptrs[sizeof...(P) > 0 ? sizeof...(P) : 1] = {static_cast<void *>(&std::get<I>(vals))...};
    return hipLaunchKernel(fn, grid, block, ptrs, shmem, stream);
}
template <typename... P, typename... A>
void launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t shmem, hipStream_t stream, A &&...args) {
    static_assert(sizeof...(P) == sizeof...(A), "kernel argument count");
    std::tuple<std::decay_t<P>...> vals(static_cast<std::decay_t<P>>(args)...);
    const hipError_t e = launch_packed(reinterpret_cast<const void *>(kernel), grid, block, shmem, stream, vals,
                                       std::index_sequence_for<P...>{});
    if (e != hipSuccess && launch_error() == hipSuccess) launch_error() = e;
}

// QIM_OK, or QIM_ERR_LAUNCH naming `what` and the first failed launch of this
// entry point (whose error is then cleared from HIP's per-thread state, so it
// is reported once, here).
int check_launch(const char *what);

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }

// Whether the bf16 rows of out, (M, N), share memory with the rows of t, (M, W): ranges that meet, other than
// other columns of one buffer.
inline bool rows_share(const void *out, int64_t ldo, int64_t N, const void *t, int64_t ldt, int64_t W, int64_t M) {
    const int64_t d = (int64_t)((intptr_t)t - (intptr_t)out) / 2;  // both 16-byte aligned
    if (d >= (M - 1) * ldo + N || -d >= (M - 1) * ldt + W) return false;
    if (M == 1 || ldt != ldo) return true;
    const int64_t col = (d % ldo + ldo) % ldo;
    return col < N || col + W > ldo;
}

// Whether the rows of out, (M, N), share memory with n vectors of W values, `step` elements apart (0: one for all; NULL: none); all in
// elements of two bytes.
inline bool rows_share_vectors(const void *out, int64_t ldo, int64_t N, int64_t M, const void *v, int64_t step, int64_t n, int64_t W) {
    if (!v) return false;
    if (step == 0) n = 1;
    const int64_t d = (int64_t)((intptr_t)v - (intptr_t)out) / 2, end = (M - 1) * ldo + N;  // both even
    if (d >= end || -d >= (n - 1) * step + W) return false;
    for (int64_t i = 0; i < n; ++i) {
        const int64_t a = d + i * step;
        if (a + W <= 0 || a >= end) continue;
        const int64_t r = a <= 0 ? 0 : a / ldo;  // the last row that starts at or before the vector; the next one may start inside
        if (a - r * ldo < N || (r + 1 < M && (r + 1) * ldo < a + W)) return true;
    }
    return false;
}

// Whether two ranges of bytes meet.
inline bool bytes_share(const void *a, int64_t na, const void *b, int64_t nb) {
    const intptr_t p = (intptr_t)a, q = (intptr_t)b;
    return p < q + nb && q < p + na;
}

// Compute units of the current device, cached per device (0 if unknown).
int device_cus();

// Lets kernel `fn` use `bytes` of dynamic LDS on the current device (HIP
// needs this above 64 KiB).  `done` is the caller's per-device record, so
// the attribute is set once per device and kernel.  QIM_OK, or
// QIM_ERR_LAUNCH with a message naming `who`.
constexpr int QIM_MAX_DEVICES = 64;
int reserve_lds(const void *fn, int bytes, std::atomic<bool> (&done)[QIM_MAX_DEVICES], const char *who);

}  // namespace qim

#define QIM_REQUIRE(cond, code, ...)                 \
    do {                                             \
        if (!(cond)) return ::qim::fail((code), __VA_ARGS__); \
    } while (0)
