// What the translation units of the torch extension share.
#pragma once

#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "../../include/pcfg_nat_hip.h"

inline void check_rc(int rc) { TORCH_CHECK(rc == PCFGNAT_OK, pcfgnat_last_error()); }

inline void *stream_of(const at::Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline void need_gpu(const char *who, std::initializer_list<const at::Tensor *> ts) {
    const at::Tensor *first = nullptr;
    for (const at::Tensor *t : ts) {
        if (t == nullptr || !t->defined()) continue;
        TORCH_CHECK(t->is_cuda(), who, ": expected tensors on the GPU, got a ", t->device().type(), " tensor");
        if (first == nullptr) first = t;
        TORCH_CHECK(t->device() == first->device(), who, ": tensors are on different devices (", first->device(), " vs ", t->device(), ")");
    }
}

// torch_ext_vocab.cpp
void register_vocab_ops(pybind11::module_ &m);
