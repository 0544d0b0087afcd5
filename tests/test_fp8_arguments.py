"""Argument checks of the 8-bit entry points, through the C ABI with host addresses (every call here is refused before anything is
launched) and through Python with CPU tensors."""
import ctypes

import pytest
import torch

from piper_amd import _lib, functional as F_, ops

ARG, SHAPE, ALIGN, UNSUPPORTED = -1, -2, -3, -5


@pytest.fixture()
def p():
    buf = ctypes.create_string_buffer(1 << 12)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    yield at
    del buf


def test_quantize(p):
    lib = _lib.load()
    rows = lib.pk_fp8_quantize_rows
    assert rows(p, 7, None, 1, p, p, 1, 128, None) == ARG
    assert rows(p, 1, None, 0, p, p, 1, 128, None) == ARG
    assert rows(p, 1, None, 1, p, p, -1, 128, None) == ARG
    assert rows(p, 1, None, 1, p, p, 1, 0, None) == ARG
    assert rows(None, 1, None, 1, p, p, 1, 128, None) == ARG
    assert rows(p, 1, None, 1, p + 4, p, 1, 128, None) == ALIGN
    assert rows(p, 1, None, 1, p, p, 2 ** 31, 128, None) == SHAPE
    assert rows(p, 1, None, 1, p, p, 2 ** 30, 1024, None) == SHAPE
    assert rows(None, 1, None, 1, None, None, 0, 128, None) == 0

    def weights(count=1, w=p, dtype=1, q=p, t=p, sc=p, E=1, N=1, K=1):
        at = lambda v: (ctypes.c_void_p * 4)(*[v] * 4)  # noqa: E731
        size = lambda v: (ctypes.c_int64 * 4)(*[v] * 4)  # noqa: E731
        return lib.pk_fp8_quantize_weights(count, at(w), dtype, at(q), at(t), at(sc), E, size(N), size(K), None)

    assert [weights(E=-1), weights(N=0), weights(K=0), weights(dtype=2), weights(w=None), weights(q=None), weights(sc=None), weights(count=-1),
            weights(count=4)] == [ARG] * 9
    assert [weights(q=p + 8), weights(t=p + 8)] == [ALIGN] * 2
    assert [weights(E=2 ** 31), weights(E=2 ** 20, N=2 ** 18), weights(E=2 ** 29, N=256, K=256), weights(count=3, E=2 ** 30), weights(N=2 ** 31)] == [SHAPE] * 5
    assert weights(E=0, w=None) == 0 and weights(count=0) == 0 and lib.pk_fp8_quantize_weights(1, None, 1, None, None, None, 1, None, None, None) == ARG


def test_products(p):
    lib = _lib.load()
    assert lib.pk_fp8_plan(p, 0, 0, 8, p, None) == ARG and lib.pk_fp8_plan(None, 0, 4, 8, p, None) == ARG and lib.pk_fp8_plan(p, 0, 4, -1, p, None) == ARG
    assert lib.pk_fp8_plan(p, 0, 1025, 8, p, None) == SHAPE and lib.pk_fp8_plan(p, 0, 4, 8, p + 4, None) == ALIGN
    assert lib.pk_fp8_plan_bytes(-1, 4) < 0 and lib.pk_fp8_plan_bytes(8, 0) < 0 and lib.pk_fp8_plan_bytes(8, 1025) < 0
    assert lib.pk_fp8_plan_bytes(1000, 6) == 4 * (8 + 8 * (1000 // 128 + 6)) and lib.pk_fp8_plan_bytes(0, 7) == 4 * 16

    def calls(A, H, I, E, q=p):
        yield lib.pk_fp8_gate_up(q, p, p, p, p, p, p, p, p, p, p, A, H, I, E, None)
        yield lib.pk_fp8_down(q, p, p, p, p, p, A, H, I, E, None)
        yield lib.pk_fp8_dgrad_dh(q, p, p, p, p, p, p, p, p, p, p, p, p, p, A, H, I, E, None)
        yield lib.pk_fp8_dgrad_dx(q, p, p, p, p, p, p, p, p, p, A, H, I, E, None)

    for A, H, I, E, want in ((-1, 128, 128, 1, ARG), (1, 0, 128, 1, ARG), (1, 128, 0, 1, ARG), (1, 128, 128, 0, ARG), (1, 8193, 128, 1, SHAPE),
                             (1, 128, 4097, 1, SHAPE), (1, 128, 128, 1025, SHAPE), (2 ** 31, 128, 128, 1, SHAPE), (2 ** 20, 8192, 128, 1, SHAPE),
                             (0, 128, 128, 1, 0)):
        assert list(calls(A, H, I, E)) == [want] * 4, (A, H, I, E)
    assert list(calls(1, 128, 128, 1, None)) == [ARG] * 4
    assert list(calls(1, 128, 128, 1, p + 8)) == [ALIGN] * 4

    def dh_t(ldt, H=256, I=256, A=10, q=p):
        return lib.pk_fp8_dgrad_dh_t(q, p, p, p, p, p, p, p, p, p, ldt, p, p, p, p, A, H, I, 2, None)

    enough = lib.pk_grouped_swiglu_transposed_ld(10, 256, 256, 2, _lib.PK_BF16)
    assert dh_t(enough, H=128) == SHAPE and dh_t(enough, I=384) == SHAPE and dh_t(enough - 64) == ARG and dh_t(enough + 1) == ARG
    assert dh_t(enough, q=None) == ARG and dh_t(enough, q=p + 8) == ALIGN and dh_t(enough, A=0) == 0 and dh_t(enough, A=-1) == ARG
    begin = lambda A=4, H=128, E=2, x=p, n=p, q=p, sc=p, plan=p: lib.pk_fp8_begin(x, n, 0, q, sc, plan, A, H, E, None)  # noqa: E731
    back = lambda A=4, H=128, E=2, x=p, q=p, sc=p, plan=p: lib.pk_fp8_begin_backward(x, plan, q, sc, p, A, H, E, None)  # noqa: E731
    for f in (begin, back):
        assert [f(A=-1), f(H=0), f(E=0), f(x=None), f(q=None), f(sc=None), f(plan=None)] == [ARG] * 7
        assert [f(H=8193), f(E=1025), f(A=2 ** 31), f(A=2 ** 20, H=8192)] == [SHAPE] * 4 and [f(q=p + 8), f(plan=p + 4)] == [ALIGN] * 2
    assert begin(n=None) == ARG and begin(A=0, n=None) == ARG and back(A=0) == 0
    # few rows
    few = lambda A=4, H=128, I=128, E=2, x=p, g=p, u=p, w=p: lib.pk_fp8_experts_few_rows(x, p, 0, w, p, p, p, p, p, g, u, p, p, A, H, I, E, None)  # noqa: E731
    assert few(A=-1) == ARG and few(H=0) == ARG and few(x=None) == ARG and few(g=None) == ARG and few(w=p + 8) == ALIGN and few(H=8200) == SHAPE
    assert few(A=0) == 0 and lib.pk_fp8_few_rows_pays(0, 128, 128, 4) == 0 and lib.pk_fp8_few_rows_pays(8, 0, 128, 4) == 0
    assert lib.pk_fp8_few_rows_pays(8, 2048, 768, 128) == 1 and lib.pk_fp8_few_rows_pays(32768, 2048, 768, 128) == 0
    # one of gate and up alone; scales of rows that are not words
    assert lib.pk_fp8_gate_up(p, p, p, p, p, p, p, p, None, p, p, 1, 128, 128, 1, None) == ARG
    assert lib.pk_fp8_down(p, p + 2, p, p, p, p, 1, 128, 128, 1, None) == ALIGN
    assert lib.pk_fp8_dgrad_dx(p, p, p, p + 1, p, p, p, p, p, p, 1, 128, 128, 1, None) == ALIGN


def test_adamw8(p):
    lib = _lib.load()
    how = (1e-3, 0.9, 0.95, 1e-8, 0.1)

    def flat(master=p, m=p, ms=p, grad=p, shadow=None, sd=1, n=64, step=1):
        return lib.pk_adamw8_fused(master, m, ms, p, p, grad, shadow, sd, n, *how, step, 0, 1.0, 0, None)

    assert flat(n=-1) == ARG and flat(step=0) == ARG and flat(master=None) == ARG and flat(ms=None) == ARG and flat(grad=None) == ARG
    assert flat(shadow=p, sd=9) == ARG and flat(m=p + 4) == ALIGN and flat(shadow=p + 2) == ALIGN and flat(n=2 ** 42) == SHAPE
    assert flat(n=0, master=None) == 0

    def packed(off=0, num=10, dt=1, shadow=None, sd=1, step=1, n=1, grads=True):
        ptrs = (ctypes.c_void_p * 1)(p)
        o, k = (ctypes.c_int64 * 1)(off), (ctypes.c_int64 * 1)(num)
        return lib.pk_adamw8_fused_packed(p, p, p, p, p, None, ptrs if grads else None, o, k, n, dt, shadow, sd, *how, step, 0, 1.0, 0, None)

    assert packed(off=-64) == ARG and packed(num=-1) == ARG and packed(dt=5) == ARG and packed(step=0) == ARG and packed(n=-1) == ARG
    assert packed(grads=False) == ARG and packed(off=63) == ALIGN and packed(off=32) == ALIGN and packed(shadow=p, sd=0) == UNSUPPORTED
    assert packed(num=2 ** 42) == SHAPE and packed(n=0) == 0


def test_cpu_tensors_are_refused():
    w1, w2 = torch.zeros(2, 128, 256).bfloat16(), torch.zeros(2, 256, 128).bfloat16()
    with pytest.raises(RuntimeError, match="GPU only"):
        F_.quantize_experts(w1, w2, w1)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.quantize_rows_fp8(w1[0])
    q, s = w1.to(torch.float8_e4m3fn), torch.zeros(2, 1, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    e = F_.Fp8Experts(w1, w2, w1, q, w2.to(torch.float8_e4m3fn), q, s, s.view(2, 2, 1), s)
    with pytest.raises(RuntimeError, match="GPU only"):
        F_.bmm_experts_fp8(e, w1[0], torch.tensor([64, 64]))
    m8 = ops.adamw8_state(64, "cpu")
    p = torch.zeros(64)
    how = dict(step=1, lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, seed=0)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.adamw8_fused(p, *m8, p, **how)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.adamw8_fused_packed(p, *m8, None, [p], [0], [64], **how)
