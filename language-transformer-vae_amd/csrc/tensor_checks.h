// What a call that hands raw memory to a kernel has to refuse, because the kernel would not carry it along: shared by the
// host helpers that read torch tensors.
#pragma once
#include <ATen/TracerMode.h>
#include <ATen/core/Tensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

// whether operators are being recorded rather than run (torch.jit.trace, make_fx, fake tensors): the record would hold the
// allocations of a call and not its kernels
inline bool being_traced() {
    using Modes = c10::impl::TorchDispatchModeTLS;
    using Key = c10::impl::TorchDispatchModeKey;
    if (at::tracer::impl::is_dispatch_enabled()) return true;
    return Modes::any_modes_set() && (Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL));
}

// why the memory of a tensor is not all there is to it, or NULL
inline const char* more_than_memory(const at::Tensor& t) {
    if (t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper})))
        return "is wrapped by a torch.func transform: there are no such transforms of this call";
    if (t._fw_grad(/*level=*/0).defined())
        return "carries a tangent: there are no forward-mode derivatives of this call";
    return nullptr;
}
