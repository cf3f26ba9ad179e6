"""Argument checks of the training-step operators (include/msccl_amd_ops.h), without a GPU: every call
here is refused before any device call.  Device addresses are made up and never followed."""
import ctypes

import pytest
import torch

import msccl_amd as M
from msccl_amd import ops

BAD = 4  # ncclInvalidArgument
F16, F32, BF16, I32, I64 = M.FLOAT16, M.FLOAT32, M.BFLOAT16, M.INT32, M.INT64
A = 1 << 20  # an aligned address


def square_create(n=2, type=F32, data=(A, A), counts=(5, 6), device=A, nbytes=1 << 16, plan=True):
    L = ops._lib()
    h = ctypes.c_void_p()
    d = (ctypes.c_void_p * max(1, len(data)))(*data) if data is not None else None
    c = (ctypes.c_size_t * max(1, len(counts)))(*counts) if counts is not None else None
    rc = L.mscclAmdSquareSumCreate(ctypes.byref(h) if plan else None, d, c, n, type, device, nbytes, None)
    assert not h
    return rc


@pytest.mark.parametrize("kw", [dict(plan=False), dict(type=M.INT32), dict(type=M.FLOAT64), dict(type=77), dict(type=-1),
                                dict(data=None), dict(counts=None), dict(device=None), dict(device=A + 4),
                                dict(nbytes=8), dict(data=(A, None)), dict(data=(A, A + 2)), dict(type=BF16, data=(A, A + 1)),
                                dict(n=1 << 21), dict(counts=(5, 1 << 62))])
def test_square_sum_create_refuses(kw):
    assert square_create(**kw) == BAD


def test_square_sum_refuses_bad_plan():
    L = ops._lib()
    junk = ctypes.create_string_buffer(256)
    for h in (None, ctypes.addressof(junk)):
        assert L.mscclAmdSquareSum(h, A, A, 1 << 20, None) == BAD
        assert L.mscclAmdSquareSumWorkspace(h) == 0
    assert L.mscclAmdSquareSumDestroy(None) == 0
    assert L.mscclAmdSquareSumDestroy(ctypes.addressof(junk)) == BAD


TENSOR_FIELDS = ("param", "grad", "master", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "count",
                 "weight_decay", "lr_scale")


def adamw_create(tensor=None, n=1, paramType=F32, gradType=F32, bits=32, step=7 * A, device=8 * A, nbytes=1 << 16, plan=True,
                 second=None):
    L = ops._lib()
    rows = b""
    for over in (tensor or {}, (tensor or {}) if second is None else second):
        o = 4096 * len(rows)
        base = dict(param=A + o, grad=2 * A + o, exp_avg=3 * A + o, exp_avg_sq=4 * A + o, count=10, lr_scale=1.0, weight_decay=0.0)
        if bits == 8:
            base |= dict(exp_avg_scale=5 * A + o, exp_avg_sq_scale=6 * A + o)
        rows += ops._TENSOR.pack(*[(base | over).get(f) or 0 for f in TENSOR_FIELDS])
    h = ctypes.c_void_p()
    rc = L.mscclAmdAdamWCreate(ctypes.byref(h) if plan else None, rows, n, paramType, gradType, bits, step, device, nbytes, None)
    assert not h
    return rc


@pytest.mark.parametrize("kw", [
    dict(plan=False), dict(paramType=I32), dict(gradType=M.FLOAT64), dict(bits=16), dict(bits=4), dict(step=None),
    dict(step=A + 4), dict(device=None), dict(device=A + 4), dict(nbytes=64), dict(n=1 << 21),
    dict(tensor=dict(param=None)), dict(tensor=dict(grad=None)), dict(tensor=dict(exp_avg=None)),
    dict(tensor=dict(exp_avg_sq=None)), dict(bits=8, tensor=dict(exp_avg_scale=None)),
    dict(bits=8, tensor=dict(exp_avg_sq_scale=None)), dict(tensor=dict(exp_avg_scale=A)),
    dict(tensor=dict(master=9 * A)),                                    # a copy of 32-bit weights
    dict(n=2, paramType=BF16, tensor=dict(master=9 * A), second=dict()),  # only some have copies
    dict(n=2, second=dict(param=A)), dict(n=2, second=dict(exp_avg=3 * A + 36)),   # a tensor twice, one in another's end
    dict(tensor=dict(exp_avg=A + 16)), dict(tensor=dict(grad=A + 20)), dict(tensor=dict(grad=7 * A)),
    dict(bits=8, tensor=dict(exp_avg_sq_scale=5 * A)), dict(n=2, second=dict(grad=4 * A - 4)),
    dict(tensor=dict(param=A + 2)), dict(gradType=F16, tensor=dict(grad=A + 1)), dict(tensor=dict(exp_avg=A + 1)),
    dict(paramType=F16, tensor=dict(master=A + 2)), dict(bits=8, tensor=dict(exp_avg_scale=A + 2)),
    dict(tensor=dict(weight_decay=float("nan"))), dict(tensor=dict(lr_scale=float("inf"))),
    dict(tensor=dict(count=1 << 62))])
def test_adamw_create_refuses(kw):
    assert adamw_create(**kw) == BAD


def test_adamw_refuses_bad_plan():
    L = ops._lib()
    junk = ctypes.create_string_buffer(256)
    for h in (None, ctypes.addressof(junk)):
        assert L.mscclAmdAdamWStep(h, 1e-3, None, 0.9, 0.99, 1e-8, 1.0, None, 0.0, None) == BAD
        assert L.mscclAmdAdamWSetGrads(h, None, 0, None) == BAD
    assert L.mscclAmdAdamWDestroy(None) == 0
    assert L.mscclAmdAdamWDestroy(ctypes.addressof(junk)) == BAD


FIELDS = ("logits", "type", "tokens", "experts", "logit_stride", "index", "index_type", "top_k", "index_stride", "valid", "score")


def router(**kw):
    base = dict(logits=A, type=F32, tokens=10, experts=8, logit_stride=8, index=A, index_type=I32, top_k=2,
                index_stride=2, valid=None, score=0)
    return ops._ROUTER.pack(*[(base | kw)[f] or 0 for f in FIELDS])


BAD_ROUTERS = [dict(type=I32), dict(type=M.FLOAT64), dict(score=2), dict(score=-1), dict(experts=0), dict(experts=1025),
               dict(top_k=0), dict(top_k=9), dict(tokens=(1 << 30) + 1), dict(tokens=1 << 30, top_k=1024, experts=1024), dict(logit_stride=7), dict(logit_stride=1 << 40),
               dict(logits=None), dict(logits=A + 2), dict(type=BF16, logits=A + 1)]


@pytest.mark.parametrize("kw", BAD_ROUTERS + [dict(index=None), dict(index_type=F32), dict(index_stride=1), dict(index=A + 2),
                                              dict(index_type=I64, index=A + 4), dict(index_stride=1 << 40)])
def test_balance_stats_refuses(kw):
    assert ops._lib().mscclAmdBalanceStats(router(**kw), A, A, A, 1 << 30, None) == BAD


def test_balance_stats_refuses_outputs():
    L, r = ops._lib(), router(tokens=50000)
    need = L.mscclAmdBalanceWorkspace(50000, 8)
    assert need > 0 and L.mscclAmdBalanceWorkspace(10, 8) == 0
    for args in [(None, A, A, need), (A, None, A, need), (A, A, None, need), (A, A, A, need - 1), (A + 4, A, A, need),
                 (A, A + 2, A, need), (A, A, A + 2, need)]:
        assert L.mscclAmdBalanceStats(r, *args, None) == BAD
    assert L.mscclAmdBalanceStats(None, A, A, A, need, None) == BAD
    assert L.mscclAmdBalanceWorkspace(10, 0) == 0 and L.mscclAmdBalanceWorkspace(10, 1025) == 0
    assert L.mscclAmdBalanceWorkspace((1 << 30) + 1, 8) == 0


@pytest.mark.parametrize("args", [(None, A, 8, 2, 1.0, A), (A, None, 8, 2, 1.0, A), (A, A, 8, 2, 1.0, None), (A, A, 0, 1, 1.0, A),
                                  (A, A, 1025, 1, 1.0, A), (A, A, 8, 0, 1.0, A), (A, A, 8, 9, 1.0, A),
                                  (A, A, 8, 2, float("nan"), A), (A + 4, A, 8, 2, 1.0, A), (A, A + 1, 8, 2, 1.0, A),
                                  (A, A, 8, 2, 1.0, A + 2)])
def test_balance_loss_refuses(args):
    assert ops._lib().mscclAmdBalanceLoss(*args, None) == BAD


@pytest.mark.parametrize("kw", BAD_ROUTERS)
def test_balance_backward_refuses(kw):
    assert ops._lib().mscclAmdBalanceBackward(router(**kw), A, 1.0, None, 2 * A, 8, 0, None) == BAD


@pytest.mark.parametrize("args", [(None, 1.0, None, 2 * A, 8, 0), (A + 4, 1.0, None, 2 * A, 8, 0), (A, float("inf"), None, 2 * A, 8, 0),
                                  (A, 1.0, A + 2, 2 * A, 8, 0), (A, 1.0, None, None, 8, 0), (A, 1.0, None, 2 * A + 2, 8, 0),
                                  (A, 1.0, None, 2 * A, 7, 0), (A, 1.0, None, 2 * A, 1 << 40, 0),
                                  (A, 1.0, None, A, 8, 1), (A, 1.0, None, A, 9, 0)])
def test_balance_backward_refuses_outputs(args):
    assert ops._lib().mscclAmdBalanceBackward(router(), *args, None) == BAD


def test_python_refuses_host_tensors():
    x = torch.zeros(4)
    with pytest.raises(ValueError):
        ops.SquareSum([x])
    with pytest.raises(ValueError):
        ops.SquareSum([])
    m, v = ops.adamw_state(x)
    with pytest.raises(ValueError):
        ops.AdamW([x], [x], [m], [v], torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.AdamW([], [], [], [], torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.balance_stats(torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.balance_backward(torch.zeros(4, 8), torch.zeros(9, dtype=torch.int64), 2)
    with pytest.raises(ValueError):
        ops.balance_loss(torch.zeros(9, dtype=torch.int64), torch.zeros(8), 2)
    with pytest.raises(ValueError):
        ops.balance_all_reduce([], [], [])
    with pytest.raises(ValueError):
        ops.sharded_step([], [], [], [], [], [], 1e-3)
    with pytest.raises(ValueError):
        ops.adamw_state(x, bits=4)


def test_states_and_their_values():
    x = torch.zeros(300)
    assert [t.shape[0] for t in ops.adamw_state(x)] == [300, 300]
    m, v, ms, vs = ops.adamw_state(x, bits=8)
    assert m.dtype == v.dtype == torch.float8_e4m3fn and ms.numel() == vs.numel() == 2
    assert ops.dequantize_state(m, ms).abs().max() == 0
    code = torch.full((300,), 2.0).to(torch.float8_e4m3fn)
    scale = torch.tensor([0.5, 3.0])
    assert ops.dequantize_state(code, scale).tolist() == [1.0] * 256 + [6.0] * 44
    assert ops.dequantize_state(code, scale, second=True).tolist() == [1.0] * 256 + [36.0] * 44


def test_router_struct_is_the_headers():
    """The packed router against the C compiler's layout of mscclAmdRouter_t."""
    class Router(ctypes.Structure):
        _fields_ = [("logits", ctypes.c_void_p), ("type", ctypes.c_int), ("tokens", ctypes.c_size_t),
                    ("experts", ctypes.c_size_t), ("logit_stride", ctypes.c_size_t), ("index", ctypes.c_void_p),
                    ("index_type", ctypes.c_int), ("top_k", ctypes.c_size_t), ("index_stride", ctypes.c_size_t),
                    ("valid", ctypes.c_void_p), ("score", ctypes.c_int)]
    values = list(range(101, 112))
    raw = ops._ROUTER.pack(*values)
    r = Router.from_buffer_copy(raw.ljust(ctypes.sizeof(Router), b"\0"))
    assert [getattr(r, f) for f in FIELDS] == values


def test_packed_structs_have_the_headers_sizes(tmp_path):
    """Sizes and offsets of the packed argument structs as the C compiler sees them."""
    import os
    import shutil
    import subprocess
    if not shutil.which("gcc"):
        pytest.skip("gcc missing")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src, exe = tmp_path / "s.c", str(tmp_path / "s")
    src.write_text("""#include <stdio.h>
#include "msccl_amd_ops.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu\\n", sizeof(mscclAmdAdamWTensor_t), offsetof(mscclAmdAdamWTensor_t, lrScale),
         offsetof(mscclAmdRouter_t, score), offsetof(mscclAmdRouter_t, topK), offsetof(mscclAmdAdamWTensor_t, count));
  return 0;
}
""")
    subprocess.run(["gcc", "-Wall", "-Werror", "-I" + os.path.join(root, "include"), "-I/opt/rocm/include",
                    "-D__HIP_PLATFORM_AMD__", str(src), "-o", exe], check=True, capture_output=True, text=True)
    got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ops._TENSOR.size, ops._TENSOR.size - 8, ops._ROUTER.size - 4, 56, 56]


def test_adamw_set_rounding_refuses_bad_plan():
    L = ops._lib()
    junk = ctypes.create_string_buffer(256)
    for h in (None, ctypes.addressof(junk)):
        assert L.mscclAmdAdamWSetRounding(h, 1, 0) == BAD


def test_adamw_check_is_the_steps():
    """The numbers that a step refuses, without a plan; a chain of collectives asks before its first."""
    L = ops._lib()
    good = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, scale=0.5, norm=0.0)
    check = lambda **kw: L.mscclAmdAdamWCheck(*(good | kw).values())  # noqa: E731
    for kw in (dict(), dict(lr=0.0), dict(lr=-1.0), dict(beta1=0.0, beta2=0.0), dict(eps=0.0), dict(norm=1.0), dict(norm=float("inf"))):
        assert check(**kw) == 0, kw
    nan, inf = float("nan"), float("inf")
    for kw in (dict(lr=nan), dict(lr=inf), dict(beta1=1.0), dict(beta2=1.0), dict(beta1=-0.1), dict(beta2=nan), dict(eps=-1.0),
               dict(eps=1e-40), dict(eps=inf), dict(scale=0.0), dict(scale=-1.0), dict(scale=1e39), dict(scale=nan), dict(norm=-1.0),
               dict(norm=nan)):
        assert check(**kw) == BAD, kw


@pytest.mark.parametrize("beta,rc", [(1 - 2.0 ** -24, 0), (1 - 2.0 ** -25, BAD), (1 - 1e-9, BAD), (1 - 1e-16, BAD)])
def test_adamw_refuses_betas_that_are_one_in_32_bits(beta, rc):
    L = ops._lib()
    assert L.mscclAmdAdamWCheck(1e-3, beta, 0.999, 1e-8, 1.0, 0.0) == rc
    assert L.mscclAmdAdamWCheck(1e-3, 0.9, beta, 1e-8, 1.0, 0.0) == rc


def test_one_tensor_for_each_version_counter():
    flats = [torch.zeros(16) for _ in range(200)]
    views = [f[4 * i:4 * i + 4] for f in flats for i in range(3)]
    whole = [torch.zeros(3) for _ in range(5)]
    del flats   # (the views keep their bases)
    got = ops._versions(views + whole + whole)
    assert len(got) == 205
    before = [t._version for t in views + whole]
    ops._changed(got)
    assert [t._version for t in views + whole] == [v + 1 for v in before]
