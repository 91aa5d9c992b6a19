// What the checked entry points of the device operators share: errors, the
// device of a call, alignments and the size of a launch.
#pragma once

#include <initializer_list>
#include <string>

#include "meshgpt_types.hpp"
#include "operators.hpp"

namespace meshgpt {

inline void check(hipError_t e, const char *what) {
    if (e == hipSuccess) return;
    (void)hipGetLastError();  // reported here
    throw Error(std::string(what) + ": " + hipGetErrorString(e), e == hipErrorOutOfMemory ? kOutOfMemory : kDeviceError);
}

inline void require(bool ok, const char *message) {
    if (!ok) throw Error(message);
}

// `device` is the current device while this lives.  What earlier calls left as
// the thread's last error is not this call's.
class OnDevice {
  public:
    explicit OnDevice(int device) {
        int count = 0;
        check(hipGetDeviceCount(&count), "hipGetDeviceCount");
        if (device < 0 || device >= count) throw Error("invalid device ordinal", kDeviceError);
        check(hipGetDevice(&caller_), "hipGetDevice");
        switched_ = caller_ != device;
        if (switched_) check(hipSetDevice(device), "hipSetDevice");
        (void)hipGetLastError();
    }
    ~OnDevice() {
        if (switched_) (void)hipSetDevice(caller_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;

  private:
    int caller_ = 0;
    bool switched_ = false;
};

inline void check_type(Type type) {
    require(type == Type::F32 || type == Type::F16 || type == Type::BF16, "unknown element type code");
}

inline bool aligned_to(int bytes, const void *p, const Strides &s, Type type) {
    const int64_t size = int64_t(type_size(type));
    bool ok = reinterpret_cast<uintptr_t>(p) % size_t(bytes) == 0;
    for (int64_t v : s.s) ok = ok && v % bytes * size % bytes == 0;
    return ok;
}
// 16, 4, or 0 for less.
inline int alignment(const void *k, const Strides &ks, const void *v, const Strides &vs, Type type) {
    for (int bytes : {16, 4})
        if (aligned_to(bytes, k, ks, type) && aligned_to(bytes, v, vs, type)) return bytes;
    return 0;
}

inline void check_aligned(const void *p, Type type, const char *message) {
    require(reinterpret_cast<uintptr_t>(p) % type_size(type) == 0, message);
}

// Of 32-bit values, null where there are none: scalar loads drop an address's last bits.
inline void check_words(std::initializer_list<const void *> words, const char *message) {
    for (const void *p : words) require(reinterpret_cast<uintptr_t>(p) % 4 == 0, message);
}

// A launch counts its threads, 256 a workgroup, in 32 bits.
inline void check_grid(double workgroups) {
    require(workgroups < double(1u << 24), "the call is too large for one launch");
}

}  // namespace meshgpt
