// The operators' host side (qxg_ops.hip) alone, with a HIP runtime and launchers that only write down what is asked of them: for
// test_ops_host.py, on the CPU.
#include "../qx-mini-c_amd/csrc/qxg_ops.hip"

extern "C" {
struct Seen {
    int last;          // the runtime's last error
    int fail;          // what the launchers end with
    int unknown;       // pointers are not known to the runtime
    int device, launches, waits, waits_that_fail;
    uint32_t wide, splits, tiles, wgs, kept, packed;   // of the last tree
} seen;

static hipError_t note(int e) {
    if (e) seen.last = e;
    return (hipError_t)e;
}
hipError_t hipGetLastError(void) { const int e = seen.last; seen.last = 0; return (hipError_t)e; }
hipError_t hipPeekAtLastError(void) { return (hipError_t)seen.last; }
hipError_t hipGetDevice(int *d) { *d = seen.device; return hipSuccess; }
hipError_t hipSetDevice(int d) { seen.device = d; return hipSuccess; }
hipError_t hipPointerGetAttributes(hipPointerAttribute_t *at, const void *) {
    if (seen.unknown) return note(hipErrorInvalidValue);
    at->type = hipMemoryTypeDevice;
    at->device = 0;
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { ++seen.waits; return note(seen.waits_that_fail); }
const char *hipGetErrorString(hipError_t e) { return e == hipErrorInvalidConfiguration ? "configuration" : e == hipErrorUnknown ? "unknown" : "other"; }
}

static hipError_t launched() { ++seen.launches; return note(seen.fail); }
int qxg_ctx_device(const qxg_ctx *) { return 0; }
hipError_t qxa_launch(const QxaArgs &A, hipStream_t) {
    seen.wide = A.wide; seen.splits = A.splits; seen.tiles = A.tiles; seen.wgs = A.wgs; seen.kept = A.scores != nullptr; seen.packed = A.pack != nullptr;
    return launched();
}
hipError_t qxe_launch_select(const qxg_kv_select_args &, hipStream_t) { return launched(); }
hipError_t qxe_launch_compact(const QxeCompact &, hipStream_t) { return launched(); }
hipError_t qxs_launch(const QxsArgs &, hipStream_t) { return launched(); }
