// The host's pow in stream order (host_pow.h): pinned staging and the host function.
#include "host_pow.h"
#include <map>
#include <mutex>
#include <new>
#include <utility>

namespace samx {
namespace {

struct Job {
    double* x;
    int64_t n;
    double y;
    bool once;      // an eager call's: it ends with its run (a captured graph runs its own any number of times)
};

void run_job(void* p) {
    Job* j = (Job*)p;
    host_pow_values(j->x, j->n, j->y);
    if (j->once) delete j;
}

struct Slot {
    double* x = nullptr;
    int64_t cap = 0;
    int dev = -1;
    hipEvent_t done = nullptr;
    bool taken = false, used = false;
};

constexpr int kSlots = 64;
constexpr int64_t kSlotMin = 4096, kChunk = int64_t(1) << 20;   // doubles

std::mutex mu;
Slot slots[kSlots];
// Memory of captured calls, carved from chunks that eager calls allocate (nothing may be allocated under capture) and
// held until the process ends.
double* chunk = nullptr;
int64_t chunk_left = 0;
struct Held { double* x; int64_t cap; };
std::map<std::pair<int, const void*>, Held>* held = nullptr;

int capturing(hipStream_t st, bool* yes) {
    hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
    SAMX_CHECK_HIP(hipStreamIsCapturing(st, &s));
    *yes = s == hipStreamCaptureStatusActive;
    return SAMX_OK;
}

// (*x stays as it was where there is no memory: what is left of a chunk goes on being given out)
int pinned(int64_t n, double** x) {
    void* got = nullptr;
    SAMX_CHECK_HIP(hipHostMalloc(&got, (size_t)n * sizeof(double), hipHostMallocPortable));
    *x = (double*)got;
    return SAMX_OK;
}

}  // namespace

void host_pow_values(double* x, int64_t n, double y) {
    for (int64_t i = 0; i < n; ++i) x[i] = pow(x[i], y);
}

int host_pow_stage(const void* owner, int64_t n, hipStream_t st, PowStage* s) {
    bool cap = false;
    if (int rc = capturing(st, &cap)) return rc;
    int dev = 0;
    SAMX_CHECK_HIP(hipGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (cap) {
        if (!held) held = new (std::nothrow) std::map<std::pair<int, const void*>, Held>();
        if (!held) return fail(SAMX_ERR_WORKSPACE, "host pow: out of host memory");
        Held* at = nullptr;
        try {
            at = &(*held)[std::make_pair(dev, owner)];
        } catch (const std::bad_alloc&) {
            return fail(SAMX_ERR_WORKSPACE, "host pow: out of host memory");
        }
        Held& h = *at;
        if (h.cap < n) {
            if (chunk_left < n)
                return fail(SAMX_ERR_WORKSPACE, "host pow: no pinned memory left for a captured call of %lld values: make "
                            "the same call once outside the capture first", (long long)n);
            h.x = chunk;
            h.cap = n;
            chunk += n;
            chunk_left -= n;
        }
        s->x = h.x;
        s->slot = -1;
        return SAMX_OK;
    }
    // room for the captured rows of a launch (fewer where they are large)
    const int64_t most = 2 * n > (int64_t(1) << 23) ? 2 * n : int64_t(1) << 23;
    const int64_t want = 32 * n < kChunk ? kChunk : 32 * n < most ? 32 * n : most;
    if (chunk_left < want / 2) {
        if (int rc = pinned(want, &chunk)) return rc;
        chunk_left = want;
    }
    int pick = -1, fresh = -1;
    for (int i = 0; i < kSlots && pick < 0; ++i) {
        Slot& t = slots[i];
        if (!t.x) { if (fresh < 0) fresh = i; continue; }
        if (t.taken || t.dev != dev || t.cap < n) continue;
        if (t.used && hipEventQuery(t.done) != hipSuccess) { (void)hipGetLastError(); continue; }
        pick = i;
    }
    if (pick < 0 && fresh < 0) {   // every slot is in flight, another device's or too small: wait for one and renew it
        for (int i = 0; i < kSlots && pick < 0; ++i)
            if (!slots[i].taken && slots[i].dev == dev) pick = i;
        if (pick < 0) return fail(SAMX_ERR_WORKSPACE, "host pow: all %d staging slots are taken", kSlots);
        Slot& t = slots[pick];
        if (t.used) SAMX_CHECK_HIP(hipEventSynchronize(t.done));
        if (t.cap < n) {
            (void)hipHostFree(t.x);
            t.x = nullptr;
            t.used = false;
            fresh = pick;
            pick = -1;
        }
    }
    if (pick < 0) {
        Slot& t = slots[fresh];
        const int64_t c = n > kSlotMin ? n : kSlotMin;
        if (!t.done || t.dev != dev) {
            if (t.done) (void)hipEventDestroy(t.done);
            t.done = nullptr;
            SAMX_CHECK_HIP(hipEventCreateWithFlags(&t.done, hipEventDisableTiming));
        }
        if (int rc = pinned(c, &t.x)) { t.x = nullptr; return rc; }
        t.cap = c;
        t.dev = dev;
        t.used = false;
        pick = fresh;
    }
    slots[pick].taken = true;
    s->x = slots[pick].x;
    s->slot = pick;
    return SAMX_OK;
}

int host_pow_run(const PowStage& s, int64_t n, double y, hipStream_t st) {
    Job* j = new (std::nothrow) Job{s.x, n, y, s.slot >= 0};
    if (!j) return fail(SAMX_ERR_WORKSPACE, "host pow: out of host memory");
    const hipError_t e = hipLaunchHostFunc(st, run_job, j);
    if (e != hipSuccess) {
        delete j;
        return fail(SAMX_ERR_HIP, "hipLaunchHostFunc failed: %s", hipGetErrorString(e));
    }
    return SAMX_OK;
}

int host_pow_done(const PowStage& s, hipStream_t st) {
    if (s.slot < 0) return SAMX_OK;
    std::lock_guard<std::mutex> lock(mu);
    Slot& t = slots[s.slot];
    t.taken = false;
    t.used = true;
    SAMX_CHECK_HIP(hipEventRecord(t.done, st));
    return SAMX_OK;
}

}  // namespace samx
