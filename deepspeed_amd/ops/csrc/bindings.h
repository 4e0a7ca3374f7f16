// What the files of bindings share: the current stream, types, and the checks that
// go before every launch.
#pragma once

#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <vector>

namespace {

[[maybe_unused]] int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default:
      TORCH_CHECK(false, "unsupported dtype ", t.scalar_type());
  }
}

void* cur_stream() {
  return reinterpret_cast<void*>(c10::hip::getCurrentHIPStream().stream());
}

// A call's tensors lie on one device, the first's, and its kernels run there,
// whichever device is the current one. Pointers of another device are no error
// to a kernel: it faults on them or reads what is not its own.
struct OneDevice {
  const char* what;
  const c10::Device device;
  const c10::DeviceGuard guard;
  template <typename... Ts>
  OneDevice(const char* what_, const at::Tensor& first, const Ts&... more)
      : what(what_), device(first.device()), guard(device) {
    (check(more), ...);
  }
  void check(const at::Tensor& t) const {
    TORCH_CHECK(t.device() == device, what, ": tensors on different devices, ",
                device, " and ", t.device());
  }
  void check(const c10::optional<at::Tensor>& t) const {
    if (t.has_value() && t->defined()) check(*t);
  }
};

// q, o, do [B, S, H, D], k, v [B, S, Hkv, D] with any strides between tokens
// and heads that keep 16-byte rows: (batch, token, head) strides, in order.
struct FlashArgs {
  const char* what;       // the call that errors name
  int B, S, H, Hkv, D;
  std::vector<long long> strides;
  FlashArgs(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
            double scale, const char* what_ = "flash") : what(what_) {
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes() &&
                q.size(0) == k.size(0) && q.size(1) == k.size(1) &&
                q.size(3) == k.size(3), what, ": q [B,S,H,D], k/v [B,S,Hkv,D]");
    B = q.size(0); S = q.size(1); H = q.size(2); D = q.size(3);
    Hkv = k.size(2);
    TORCH_CHECK(D == 64 || D == 96 || D == 128, what, ": D of 64, 96 or 128");
    TORCH_CHECK(Hkv > 0 && H % Hkv == 0, what, ": H a multiple of Hkv");
    TORCH_CHECK(scale > 0, what, ": scale must be positive");
    TORCH_CHECK(q.size(1) < (1 << 30) && q.size(0) * (int64_t)H *
                ((S + 127) / 128) < (1ll << 31), what, ": size");
  }
  void add(const at::Tensor& t, const at::Tensor& like) {
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 &&
                t.sizes() == like.sizes() && t.stride(3) == 1 &&
                ((uintptr_t)t.data_ptr() & 15) == 0 &&
                t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
                t.stride(2) % 8 == 0 && t.stride(1) >= 0 &&
                t.stride(1) < (1 << 24), what, ": bf16 GPU, 16-byte rows");
    for (int d = 0; d < 3; ++d) strides.push_back(t.stride(d));
  }
};

}  // namespace
