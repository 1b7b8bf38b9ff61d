// What a kernel needs set up on a device before its first launch there (function attributes belong to a device, and one process
// may drive several), between threads: launchers run without the interpreter's lock.
#pragma once

namespace mxb {

// True where the bit of `device` is not yet in `seen` (one word for each call site).  The device is marked when the object goes,
// which is after the setup: a thread that meets another's unfinished setup does it again, which is harmless, instead of launching
// without it.  A setup that failed is not marked.
//   if (FirstOnDevice first{&seen, device}) { if (int code = first.take(set_attribute())) return code; }
class FirstOnDevice {
 public:
  FirstOnDevice(unsigned long long* seen, int device) : seen_(seen), bit_(1ull << (device & 63)) {
    needed_ = !(__atomic_load_n(seen_, __ATOMIC_ACQUIRE) & bit_);
  }
  FirstOnDevice(const FirstOnDevice&) = delete;
  FirstOnDevice& operator=(const FirstOnDevice&) = delete;
  ~FirstOnDevice() { if (needed_ && !failed_) __atomic_fetch_or(seen_, bit_, __ATOMIC_RELEASE); }
  explicit operator bool() const { return needed_; }
  // The code of one step of the setup (0: done).
  int take(int code) {
    if (code) failed_ = true;
    return code;
  }

 private:
  unsigned long long* seen_;
  unsigned long long bit_;
  bool needed_, failed_ = false;
};

}  // namespace mxb
