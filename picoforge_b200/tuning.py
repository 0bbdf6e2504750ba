"""Python plumbing (ctypes) of the operators that adapt and train a layer: low-rank adapters of many requests beside a
projection, the balance loss of a router, and their gradients (include/qwen4_moe_b200.h, csrc/adapters.cu, csrc/balance.cu).

Everything is a device pointer (an int, for instance torch's `data_ptr()`), FP32 unless said otherwise, dense unless a pitch
is given.  Calls enqueue on the stream in force and return without waiting; `TuneWork.sync` waits and raises what the kernels
found.  A torch program makes the library use its stream with `lib.qw4cu_set_stream(stream.cuda_stream or 1)`.
"""
from __future__ import annotations

import ctypes as C

from . import abi

NO_ADAPTER = 0xFFFFFFFF


class TuneWork:
    """A workspace (QW4CuTuneWork) and the calls on it.  `slots`, `rank`: adapters; `experts`: balance loss; 0 leaves a part out."""

    def __init__(self, api: abi.MoeApi, tokens: int, slots: int = 0, rank: int = 0, experts: int = 0):
        self.api, self.handle, self.error = api, C.c_void_p(), abi.Qwen4Error()
        self._err = C.byref(self.error)
        limits = abi.QW4CuTuneLimits(tokens, slots, rank, experts)
        self._check(api.lib.qw4cu_tune_work_create(C.byref(limits), C.byref(self.handle), self._err))

    def _check(self, status):
        if status:
            raise abi.MoeError(status, self.error)

    @staticmethod
    def adapters(a, b, scale, gguf_type, slots, rank, k, n) -> abi.QW4CuAdapters:
        """Pointers to A [slots, rank, k], B [slots, n, rank] (F32, F16 or BF16) and scale [slots] (or None) as one view."""
        return abi.QW4CuAdapters(a, b, scale, gguf_type, slots, rank, k, n)

    @staticmethod
    def router(experts, top_k, norm_topk_prob) -> abi.Qwen4MoeConfig:
        """What the balance loss reads of a layer's configuration."""
        return abi.Qwen4MoeConfig(experts=experts, top_k=top_k, norm_topk_prob=norm_topk_prob)

    def adapter_forward(self, adapters, x, slots, base, y, tokens, x_pitch=0, base_pitch=0, y_pitch=0):
        """y[t] = base[t] + scale B (A x[t]) with the adapter slots[t]; pitches in bytes, 0: dense."""
        k4, n4 = adapters.k * 4, adapters.n * 4
        self._check(self.api.lib.qw4cu_adapter_forward_device(
            C.byref(adapters), x, x_pitch or k4, slots, base, base_pitch or n4, y, y_pitch or n4, tokens, self.handle, self._err))

    def adapter_backward(self, adapters, x, slots, dy, base, dx, da, db, tokens, x_pitch=0, dy_pitch=0, base_pitch=0, dx_pitch=0):
        k4, n4 = adapters.k * 4, adapters.n * 4
        self._check(self.api.lib.qw4cu_adapter_backward_device(
            C.byref(adapters), x, x_pitch or k4, slots, dy, dy_pitch or n4, base, base_pitch or k4, dx, dx_pitch or k4, da, db, tokens,
            self.handle, self._err))

    def route(self, layer, adapters, x, slots, tokens, logits=None, ids=None, weights=None):
        """Routes of a `MoeLayer` with adapters (or None) beside its router; logits [tokens, experts]: what was routed."""
        self._check(self.api.lib.qw4cu_moe_route_adapted_device(
            layer.moe, x, tokens, C.byref(adapters) if adapters else None, slots, self.handle, logits, ids, weights, layer.work, self._err))

    def layer_forward(self, layer, adapters, x, slots, y, tokens, logits=None, ids=None, weights=None):
        """The whole layer on those routes."""
        self._check(self.api.lib.qw4cu_moe_forward_adapted_device(
            layer.moe, x, y, tokens, C.byref(adapters) if adapters else None, slots, self.handle, logits, ids, weights, layer.work, self._err))

    def balance_forward(self, config, logits, ids, mask, tokens, counts, prob_sums, loss, logits_pitch=0):
        self._check(self.api.lib.qw4cu_balance_forward_device(
            C.byref(config), logits, logits_pitch or config.experts * 4, ids, mask, tokens, counts, prob_sums, loss, self.handle, self._err))

    def balance_backward(self, config, logits, ids, mask, tokens, counts, loss_grad, weights_grad, grad, logits_pitch=0, grad_pitch=0):
        e4 = config.experts * 4
        self._check(self.api.lib.qw4cu_balance_backward_device(
            C.byref(config), logits, logits_pitch or e4, ids, mask, tokens, counts, loss_grad, weights_grad, grad, grad_pitch or e4,
            self.handle, self._err))

    def sync(self):
        self._check(self.api.lib.qw4cu_tune_work_sync(self.handle, self._err))

    def reset(self):
        self._check(self.api.lib.qw4cu_tune_work_reset(self.handle, self._err))

    def close(self):
        if self.handle:
            self.api.lib.qw4cu_tune_work_destroy(self.handle)
            self.handle = C.c_void_p()

    def __enter__(self):
        return self

    def __exit__(self, *_):
        self.close()

    def __del__(self):
        if getattr(self, "handle", None):
            self.close()
