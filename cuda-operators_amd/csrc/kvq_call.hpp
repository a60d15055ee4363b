// kvq_call.hpp -- what every launching entry point does around its launches:
// the device check, then (KVQ_DEBUG_SYNC) the stream's completion status.
#pragma once

#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <mutex>

namespace kvq {

// An environment switch that is on ("1", "true", "yes", "on").
inline bool env_on(const char* name) {
    const char* s = getenv(name);
    if (!s) return false;
    static const char* const kOn[] = {"1", "true", "yes", "on", "TRUE", "YES", "ON", "True", "Yes", "On"};
    for (const char* o : kOn)
        if (strcmp(s, o) == 0) return true;
    return false;
}

// KVQ_DEBUG_SYNC, read once from the environment on first use.
inline bool debug_sync() {
    static const bool on = env_on("KVQ_DEBUG_SYNC");
    return on;
}

// The library's code objects are built for gfx950 only.  Checked once per
// device before its first launch, as the reference warns once about an
// untuned architecture (kv_cache/KV_int8_split_optimized.cu:57-65); here
// another architecture cannot run the kernels at all, so the call fails with
// hipErrorInvalidDevice after one stderr line.
inline std::mutex g_arch_mutex;
inline signed char g_arch_state[64];  // 0 unknown, 1 gfx950, -1 other

inline hipError_t arch_check() {
    int dev = 0;
    hipError_t err = hipGetDevice(&dev);
    if (err != hipSuccess) return err;
    if (dev < 0 || dev >= 64) return hipErrorInvalidDevice;
    std::lock_guard<std::mutex> lock(g_arch_mutex);
    if (g_arch_state[dev] == 0) {
        hipDeviceProp_t prop;
        err = hipGetDeviceProperties(&prop, dev);
        if (err != hipSuccess) return err;
        const bool ok = strncmp(prop.gcnArchName, "gfx950", 6) == 0 &&
                        (prop.gcnArchName[6] == '\0' || prop.gcnArchName[6] == ':');
        g_arch_state[dev] = ok ? 1 : -1;
        if (!ok)
            fprintf(stderr, "[kvq] device %d is %s; libkvq is built for gfx950 (MI355X) only\n", dev,
                    prop.gcnArchName);
    }
    return g_arch_state[dev] > 0 ? hipSuccess : hipErrorInvalidDevice;
}

inline hipError_t finish_call(hipError_t err, hipStream_t stream) {
    if (err != hipSuccess || !debug_sync()) return err;
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    err = hipStreamIsCapturing(stream, &st);
    if (err != hipSuccess || st != hipStreamCaptureStatusNone) return err;
    // The launchers already returned their launch status; the caller's own
    // pending error (hipGetLastError) is left for the caller.
    return hipStreamSynchronize(stream);
}

// Every launching entry point returns through here: the device check, the
// launches, then (KVQ_DEBUG_SYNC) the stream's completion status.
template <class Launch>
hipError_t checked_call(hipStream_t stream, Launch&& launch) {
    const hipError_t err = arch_check();
    if (err != hipSuccess) return err;
    return finish_call(launch(), stream);
}

}  // namespace kvq
