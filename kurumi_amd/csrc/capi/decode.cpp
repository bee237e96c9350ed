// C entry points of one decode step on caller-owned device buffers (include/kurumi_hip.h): the block
// of arguments is checked before the backend, so that a refusal needs no GPU.
#include <cstdint>
#include <string>

#include "../../../include/kurumi_hip.h"
#include "../hip/kernels/decode.h"
#include "backend_handle.h"
#include "errors.h"

using ku::capi::guard;
using ku::capi::set_err;

namespace {

// The backend's device for the length of a call; the caller's current device afterwards.
class OnDevice {
 public:
  explicit OnDevice(ku::hipbk::Context& ctx) {
    KU_HIP(hipGetDevice(&was_));
    if (was_ != ctx.device()) {
      ctx.make_current();
      moved_ = true;
    }
  }
  ~OnDevice() {
    if (moved_) (void)hipSetDevice(was_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

 private:
  int was_ = 0;
  bool moved_ = false;
};

// `check` on the arguments, then `launch` on the backend's device and the call's stream.
template <class Args, class Check, class Launch>
int32_t on_backend(const char* name, const KuBackend* b, const Args* args, void* stream, Check&& check, Launch&& launch) {
  return guard<int32_t>(-1, [&] {
    try {
      if (!args) throw std::runtime_error("null arguments");
      check(*args);
      if (!b) throw std::runtime_error("null backend handle");
      ku::hipbk::Context& ctx = b->b->ctx();
      OnDevice on(ctx);
      launch(*args, stream ? static_cast<hipStream_t>(stream) : ctx.stream());
    } catch (const std::exception& e) {
      throw ku::Error(std::string(name) + ": " + e.what());
    }
    return 0;
  });
}

}  // namespace

extern "C" {

int32_t ku_hip_rope_freqs(size_t rot_dim, double base, uint32_t scaling, double factor, double trained_len, double low,
                          double high, double* out) {
  return guard<int32_t>(-1, [&] {
    try {
      ku::hipbk::rope_freqs(rot_dim, base, scaling, factor, trained_len, low, high, out);
    } catch (const std::exception& e) {
      throw ku::Error(std::string("ku_hip_rope_freqs: ") + e.what());
    }
    return 0;
  });
}

int32_t ku_hip_rope(const KuBackend* b, const KuHipRopeArgs* args, void* stream) {
  return on_backend("ku_hip_rope", b, args, stream, ku::hipbk::check_rope, ku::hipbk::launch_rope);
}

int32_t ku_hip_logits_adjust(const KuBackend* b, const KuHipLogitsArgs* args, void* stream) {
  return on_backend("ku_hip_logits_adjust", b, args, stream, ku::hipbk::check_logits_adjust,
                    ku::hipbk::launch_logits_adjust);
}

size_t ku_hip_sdpa_prefix_scratch(const KuHipSdpaPrefixArgs* args) {
  return guard<size_t>(SIZE_MAX, [&] {
    try {
      if (!args) throw std::runtime_error("null arguments");
      ku::hipbk::check_sdpa_prefix(*args);
      return ku::hipbk::sdpa_prefix_scratch_bytes(*args);
    } catch (const std::exception& e) {
      throw ku::Error(std::string("ku_hip_sdpa_prefix_scratch: ") + e.what());
    }
  });
}

int32_t ku_hip_sdpa_prefix(const KuBackend* b, const KuHipSdpaPrefixArgs* args, void* stream) {
  return on_backend(
      "ku_hip_sdpa_prefix", b, args, stream,
      [](const KuHipSdpaPrefixArgs& a) {
        ku::hipbk::check_sdpa_prefix(a);
        if (a.scratch && a.scratch_bytes < ku::hipbk::sdpa_prefix_scratch_bytes(a))
          throw std::runtime_error("scratch_bytes is less than ku_hip_sdpa_prefix_scratch");
      },
      [&](const KuHipSdpaPrefixArgs& a, hipStream_t s) {
        const size_t need = ku::hipbk::sdpa_prefix_scratch_bytes(a);
        void* scratch = a.scratch;
        if (need && !scratch) {
          hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
          KU_HIP(hipStreamIsCapturing(s, &st));
          if (st != hipStreamCaptureStatusNone)
            throw std::runtime_error("a captured call needs its own scratch (ku_hip_sdpa_prefix_scratch bytes)");
          scratch = b->b->workspace(ku::hipbk::HipBackend::Entry::SdpaPrefix, need);
        }
        ku::hipbk::launch_sdpa_prefix(a, scratch, s);
      });
}

}  // extern "C"
