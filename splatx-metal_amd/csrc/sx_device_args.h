// sx_device_args.h — what the entry points of the learned heads' operators (learn.cpp, linear.cpp) check their arguments
// with: types, device memory and its extents, overlaps, the queue of a call.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>
#include <vector>

#include "splatx_hip.h"
#include "sx_host.h"
#include "sx_learn.h"

namespace sxh {

constexpr size_t type_size(uint8_t t) { return t == SXH_TYPE_F32 ? 4 : 2; }

inline void need_type(const char* what, uint8_t t, const char* name) {
    if (t != SXH_TYPE_F32 && t != SXH_TYPE_BF16 && t != SXH_TYPE_F16)
        invalid(what, std::string(name) + " must be SXH_TYPE_F32, _BF16 or _F16");
}

// The device memory of a call: each range a caller names lies in an allocation of the backend's device. (A lookup is
// 0.16 us; the buffers of a network mostly lie in a few allocations of its framework's allocator, so the last eight found
// in this call are tried first.)
class DeviceMemory {
  public:
    DeviceMemory(const char* what, int device) : what_(what), device_(device) {}
    void need(const void* p, size_t bytes, size_t align, const char* name) {
        if (!p) invalid(what_, std::string("null ") + name);
        const auto at = reinterpret_cast<uintptr_t>(p);
        if (at % align) invalid(what_, std::string(name) + " is not aligned to its elements");
        for (const Range& r : found_)
            if (at >= r.base && at - r.base <= r.size && bytes <= r.size - (at - r.base)) return;
        hipPointerAttribute_t attr{};
        if (hipPointerGetAttributes(&attr, p) != hipSuccess || attr.type != hipMemoryTypeDevice || attr.device != device_) {
            (void)hipGetLastError();  // an unknown host pointer leaves an error behind; it is reported here
            invalid(what_, std::string(name) + " is not device memory of the backend's device");
        }
        hipDeviceptr_t base = nullptr;
        size_t size = 0;
        if (hipMemGetAddressRange(&base, &size, const_cast<void*>(p)) != hipSuccess || !base) {
            (void)hipGetLastError();
            invalid(what_, std::string(name) + ": the allocation holding it is unknown");
        }
        const Range r{reinterpret_cast<uintptr_t>(base), size};
        found_[next_++ % kFound] = r;
        if (at - r.base > r.size || bytes > r.size - (at - r.base))
            invalid(what_, std::string(name) + " ends outside its allocation (" + std::to_string(bytes) + " bytes needed)");
    }

  private:
    struct Range {
        uintptr_t base = 0;
        size_t size = 0;
    };
    static constexpr unsigned kFound = 8;
    const char* what_;
    int device_;
    Range found_[kFound];
    unsigned next_ = 0;
};

// Rows of `width` bytes, `stride` bytes apart.
struct Rows {
    const char* name = nullptr;
    uintptr_t at = 0;
    size_t extent = 0, width = 0, stride = 0;
};

// Whether no byte of one lies in a row of the other. Rows of one stride may lie between each other's, as the column
// ranges of one wide buffer do.
inline bool apart(const Rows& a, const Rows& b) {
    if (!a.extent || !b.extent || a.at + a.extent <= b.at || b.at + b.extent <= a.at) return true;
    if (a.stride != b.stride || !a.stride) return false;
    const Rows &lo = a.at <= b.at ? a : b, &hi = a.at <= b.at ? b : a;
    const size_t off = (hi.at - lo.at) % a.stride;
    return off >= lo.width && a.stride - off >= hi.width;
}

struct RowCheck {
    const char* what;
    DeviceMemory mem;
    int64_t rows, width;
    std::vector<Rows> in, out;

    RowCheck(const char* w, int device, int64_t r, int64_t c) : what(w), mem(w, device), rows(r), width(c) {
        if (rows < 0) invalid(what, "negative rows");
        if (width < 1 || width > (int64_t{1} << 24)) invalid(what, "width must be 1..16777216");
        in.reserve(8);
        out.reserve(4);
    }
    void add(const void* p, int64_t stride, size_t elem, const char* name, bool written) { add(p, stride, width, elem, name, written); }
    void add(const void* p, int64_t stride, int64_t width, size_t elem, const char* name, bool written) {
        if (rows == 0) return;
        if (rows > 1 && stride < width && !(stride == 0 && !written))
            invalid(what, std::string(name) + " has rows closer together than their width");
        size_t extent = 0;
        const size_t step = rows > 1 ? static_cast<size_t>(stride) * elem : 0;
        if (rows > 1 && (static_cast<uint64_t>(stride) > (uint64_t{1} << 60) ||
                         __builtin_mul_overflow(static_cast<size_t>(rows - 1), step, &extent) || extent > (size_t{1} << 60)))
            invalid(what, std::string(name) + " is larger than memory");
        extent += static_cast<size_t>(width) * elem;
        mem.need(p, extent, elem, name);
        (written ? out : in).push_back({name, reinterpret_cast<uintptr_t>(p), extent, static_cast<size_t>(width) * elem, step});
    }
    void add_flat(const void* p, int64_t n, size_t elem, const char* name, bool written) {
        if (n == 0) return;
        const size_t bytes = static_cast<size_t>(n) * elem;
        mem.need(p, bytes, elem, name);
        (written ? out : in).push_back({name, reinterpret_cast<uintptr_t>(p), bytes, bytes, 0});
    }
    void disjoint() const {
        for (size_t i = 0; i < out.size(); i++) {
            for (const Rows& r : in)
                if (!apart(out[i], r)) invalid(what, std::string(out[i].name) + " overlaps " + r.name);
            for (size_t k = 0; k < i; k++)
                if (!apart(out[i], out[k])) invalid(what, std::string(out[i].name) + " overlaps " + out[k].name);
        }
    }
};

// The backend's device as the current one, and the stream of a call; the caller's device again afterwards.
class Queue {
  public:
    Queue(sxh_backend* b, const sxh_queue* q, const char* what) : waits_(!q), stream_(q ? static_cast<hipStream_t>(q->stream) : b->stream) {
        SXH_HIP(hipGetDevice(&before_));
        if (q && q->stream) {
            int device = -1;
            if (hipStreamGetDevice(stream_, &device) != hipSuccess || device != b->device) {
                (void)hipGetLastError();
                invalid(what, "the queue's stream is not one of the backend's device");
            }
        }
        if (before_ != b->device) SXH_HIP(hipSetDevice(b->device));
        device_ = b->device;
        (void)hipGetLastError();  // what the caller's own calls left is not this call's
    }
    ~Queue() {
        if (before_ != device_) (void)hipSetDevice(before_);
    }
    hipStream_t stream() const { return stream_; }
    void done() const {
        SXH_HIP(hipGetLastError());
        if (waits_) SXH_HIP(hipStreamSynchronize(stream_));
    }

  private:
    bool waits_;
    hipStream_t stream_;
    int before_ = 0, device_ = 0;
};

inline sxk::ElemType elem(uint8_t t) { return static_cast<sxk::ElemType>(t); }

}  // namespace sxh
