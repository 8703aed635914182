// The calling thread's current device during a call.  Plain C++ over two functions, so that a host test can stand in for them.
#pragma once

// Api::get(int*) and Api::set(int) return 0 on success.  With `put_back` the device that was current before is current again
// afterwards: for calls next to another owner of the GPUs.
template <class Api>
class rg_device_scope {
  public:
    rg_device_scope(int device, bool put_back) {
        int now = -1;
        if (Api::get(&now) != 0) now = -1;
        if (now == device) return;
        failed_ = Api::set(device);
        if (put_back && now >= 0) before_ = now;
    }
    ~rg_device_scope() {
        if (before_ >= 0) Api::set(before_);
    }
    rg_device_scope(const rg_device_scope&) = delete;
    rg_device_scope& operator=(const rg_device_scope&) = delete;
    int failed() const { return failed_; }  // what Api::set returned

  private:
    int before_ = -1, failed_ = 0;
};
