"""First phases of the token-sequence operators (no GPU): exported symbols, what they accept and what they refuse, with which status.
Tensors of these tests are on the CPU, so an accepted call ends before its second phase with the binding's ValueError."""
import ctypes
import os
import re

import pytest
import torch

NULLPTR, INVALID = 161001, 161002
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def accepted(call):
    with pytest.raises(ValueError, match="cuda device"):
        call()


def refused(ops, call, text="", status=INVALID):
    with pytest.raises(ops.AclnnError) as e:
        call()
    assert e.value.status == status and text in str(e.value)


def test_library_exports_the_declared_symbols(ops):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "aclnn_sequence.h")).read()
    declared = set(re.findall(r"ACLNN_API\s+[\w\s\*]+?\b(\w+)\s*\(", text))
    assert declared == set(ops.SEQUENCE_SYMBOLS)
    handle = ctypes.CDLL(ops.LIB_PATH)
    assert not [s for s in declared if not hasattr(handle, s)]


def test_null_arguments(ops):
    n, e = ctypes.c_uint64(7), ctypes.c_void_p(None)
    L = ops.lib()
    for name in sorted(s[:-len("GetWorkspaceSize")] for s in ops.SEQUENCE_SYMBOLS if s.endswith("GetWorkspaceSize")):
        types = ops.SEQUENCE_SYMBOLS[name + "GetWorkspaceSize"][1]
        zeros = [None if t is ctypes.c_void_p else t(0) for t in types[:-2]]
        first = getattr(L, name + "GetWorkspaceSize")
        assert first(*zeros, ctypes.byref(n), ctypes.byref(e)) == NULLPTR
        assert first(*zeros, None, ctypes.byref(e)) == NULLPTR
        assert first(*zeros, ctypes.byref(n), None) == NULLPTR
        assert n.value == 7 and e.value is None
        assert getattr(L, name)(None, 0, None, None) == NULLPTR


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_norm_accepts(ops, t):
    x = torch.zeros(2, 3, 8, dtype=t)
    w = torch.ones(8, dtype=t)
    accepted(lambda: ops.residual_rms_norm(x))
    accepted(lambda: ops.residual_rms_norm(x, x, w, 0.0))
    accepted(lambda: ops.residual_rms_norm(x, x, torch.ones(8)))
    accepted(lambda: ops.residual_rms_norm(torch.zeros(8, dtype=t)))
    accepted(lambda: ops.residual_rms_norm(torch.zeros(0, 8, dtype=t)))
    accepted(lambda: ops.residual_rms_norm(x.expand(5, 2, 3, 8), None, w))
    accepted(lambda: ops.residual_rms_norm(torch.zeros(2, 8, 3, dtype=t).transpose(1, 2), None, w))
    accepted(lambda: ops.residual_rms_norm_backward(x, x, torch.zeros(2, 3), w, x))
    accepted(lambda: ops.residual_rms_norm_backward(x, x, torch.zeros(2, 3)))
    for group in (0, 32, 96, 128, 4096):
        accepted(lambda: ops.residual_rms_norm_quant(x, x, w, group=group))
        accepted(lambda: ops.residual_rms_norm_quant(x, x, w, dtype=torch.int8, group=group))


def test_norm_refuses(ops):
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    norm, quant, back = ops.residual_rms_norm, ops.residual_rms_norm_quant, ops.residual_rms_norm_backward
    refused(ops, lambda: norm(x.double(), out=x, rstd_out=x), "dtype DOUBLE")
    refused(ops, lambda: norm(torch.zeros(3, 0)), "last extent")
    refused(ops, lambda: norm(x, x.half()), "residual must have the type")
    refused(ops, lambda: norm(x, x[:1]), "residual must have the shape")
    refused(ops, lambda: norm(x, None, w[:7]), "weight must be [8]")
    refused(ops, lambda: norm(x, None, w.half()), "weight must have")
    refused(ops, lambda: norm(x, eps=-1e-6), "eps")
    refused(ops, lambda: norm(x, eps=float("nan")), "eps")
    refused(ops, lambda: norm(x, out=x[..., :7]), "y must have the shape")
    refused(ops, lambda: norm(x, out=torch.zeros(1, 3, 8).expand(2, 3, 8)), "overlap")
    refused(ops, lambda: norm(x, x, sum_out=torch.zeros(1, 1, 8).expand(2, 3, 8)), "overlap")
    refused(ops, lambda: norm(x, rstd_out=torch.zeros(2, 3, dtype=F16)), "rstd must be FLOAT")
    refused(ops, lambda: norm(x, rstd_out=torch.zeros(3, 2)), "rstd")
    refused(ops, lambda: norm(x, rstd_out=torch.zeros(3, 2).t()), "rstd must be contiguous")
    refused(ops, lambda: back(x, x, torch.zeros(2, 2), w), "rstd")
    refused(ops, lambda: back(x, x, torch.zeros(2, 3), None, grad_weight=w), "without a weight")
    refused(ops, lambda: back(x, x, torch.zeros(2, 3), w, grad_weight=w.half()), "gradWeight")
    refused(ops, lambda: back(x, x, torch.zeros(2, 3), w, x.half()), "gradSum")
    refused(ops, lambda: back(x, x, torch.zeros(2, 3), w, grad_x=torch.zeros(1, 1, 8).expand(2, 3, 8)), "overlap")
    for group in (-32, 1, 31, 48):
        refused(ops, lambda: quant(x, group=group), "group")
    refused(ops, lambda: quant(x, scales_out=torch.zeros(2, 3)), "scales")
    refused(ops, lambda: quant(x, out=torch.zeros(2, 3, 16, dtype=torch.float8_e4m3fn)[..., ::2]), "contiguous")
    with pytest.raises(ValueError, match="dtype"):
        quant(x, dtype=torch.uint8)
    with pytest.raises(ValueError, match="type"):
        quant(x, out=torch.zeros(2, 3, 8, dtype=torch.int8))


def test_rotary_accepts(ops):
    q, k, f = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16), torch.zeros(8)
    p = torch.arange(5)
    accepted(lambda: ops.rotary_embedding(q, k, p, f))
    accepted(lambda: ops.rotary_embedding(q, None, p.int().expand(2, 5), f.double(), True, scale=1.3))
    accepted(lambda: ops.rotary_embedding(q, k, p.expand(3, 2, 5), f, sections=(4, 0, 4)))
    accepted(lambda: ops.rotary_embedding_backward(q, k, p, f[:3]))
    accepted(lambda: ops.rotary_embedding(q.transpose(1, 2), None, p[:4], f))
    accepted(lambda: ops.rotary_embedding(torch.zeros(0, 5, 4, 16), None, p, f))
    accepted(lambda: ops.rotary_embedding(q[0, 0], None, p[0], f))


def test_rotary_refuses(ops):
    q, k, f, p = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16), torch.zeros(8), torch.arange(5)
    turn = ops.rotary_embedding
    refused(ops, lambda: turn(q.double(), None, p, f), "dtype DOUBLE")
    refused(ops, lambda: turn(q, k.half(), p, f), "one type")
    refused(ops, lambda: turn(q, k[:1], p, f), "leading dimensions")
    refused(ops, lambda: turn(q, k[..., :8], p, f), "dim")
    refused(ops, lambda: turn(q, k, p.to(torch.float32), f), "positions must be")
    refused(ops, lambda: turn(q, k, p, f.half()), "frequencies must be")
    refused(ops, lambda: turn(q, k, p, torch.zeros(9)), "do not fit")
    refused(ops, lambda: turn(q, k, p, torch.zeros(0)), "do not fit")
    refused(ops, lambda: turn(q, k, p, torch.zeros(16)[::2]), "contiguous")
    refused(ops, lambda: turn(q, k, p, f, scale=float("inf")), "scale")
    refused(ops, lambda: turn(q, k, p.expand(2, 2, 5), f, sections=(4, 3)), "add up")
    refused(ops, lambda: turn(q, k, p.expand(2, 2, 5), f, sections=(9, -1)), "section")
    refused(ops, lambda: turn(q, k, p.expand(3, 2, 5), f, sections=(4, 4)), "positions must be")
    refused(ops, lambda: turn(q, k, p.expand(5, 2, 5), f, sections=(2, 2, 2, 1, 1)), "sections")
    refused(ops, lambda: turn(q, k, p, f, q_out=torch.zeros(1, 1, 1, 16).expand(2, 5, 4, 16)), "overlap")
    refused(ops, lambda: turn(q, k, p, f, q_out=q[:1]), "q's shape")
    with pytest.raises(RuntimeError, match="expand"):
        turn(q, k, p[:4], f)
    with pytest.raises(ValueError, match="without k"):
        turn(q, None, p, f, k_out=k)
    with pytest.raises(RuntimeError, match="positions|strided"):
        turn(torch.zeros(2, 3, 4, 1, 8), None, torch.zeros(8, 8, 8, dtype=torch.int64)[:2, ::2, ::2][:, :3, :4], f[:4])


def test_rotary_frequencies_refuses(ops):
    make = ops.rotary_frequencies
    for how in (dict(base=1.0), dict(base=float("nan")), dict(factor=0.5), dict(scaling="wavelength", factor=2.0),
                dict(scaling="wavelength", original_length=100.0, low=4.0, high=4.0), dict(scaling="ramp", original_length=100.0, low=0.0)):
        refused(ops, lambda: make(8, device="cpu", **how))
    refused(ops, lambda: make(8, dtype=F16, device="cpu"), "out must be")
    refused(ops, lambda: make(8, out=torch.zeros(8)[::2]), "contiguous")
    with pytest.raises(ValueError, match="even"):
        make(7)
    with pytest.raises(ValueError, match="scaling"):
        make(8, scaling="none")
    accepted(lambda: make(8, device="cpu"))
    accepted(lambda: make(8, scaling="ramp", factor=4.0, original_length=100.0, low=1.0, high=32.0, dtype=torch.float64, device="cpu"))


def test_attention_accepts(ops):
    for t in (F32, F16, BF16):
        q, k = torch.zeros(2, 5, 4, 16, dtype=t), torch.zeros(2, 9, 2, 16, dtype=t)
        accepted(lambda: ops.window_attention(q, k, k, 3, 1))
        accepted(lambda: ops.window_attention(q, k, k, 2 ** 40, 2 ** 40, scale=-1.0))
        accepted(lambda: ops.window_attention(q, k[:, :0], k[:, :0], 3))
        accepted(lambda: ops.window_attention(q[:, :0], k, k, 3))
        n = torch.tensor([5, 9])
        accepted(lambda: ops.window_attention(q, k, k, 3, kv_lengths=n, q_lengths=n.int()))
        lse = torch.zeros(2, 4, 5)
        accepted(lambda: ops.window_attention_backward(q, q, k, k, q, lse, 3, 1))
        accepted(lambda: ops.window_attention_backward(q[:, :0], q[:, :0], k, k, q[:, :0], lse[..., :0].contiguous(), 3, 1))


def test_attention_refuses(ops):
    q, k, lse = torch.zeros(2, 5, 4, 16), torch.zeros(2, 9, 2, 16), torch.zeros(2, 4, 5)
    att, back = ops.window_attention, ops.window_attention_backward
    refused(ops, lambda: att(q.double(), k.double(), k.double(), 3, out=q, lse=lse), "dtype DOUBLE")
    refused(ops, lambda: att(q, k.half(), k.half(), 3), "one type")
    refused(ops, lambda: att(q, k, k[:, :8], 3), "k's shape")
    refused(ops, lambda: att(q, k[:1], k[:1], 3), "one batch")
    refused(ops, lambda: att(q, k[..., :8], k[..., :8], 3), "one dim")
    refused(ops, lambda: att(q[:, :, :3], k, k, 3), "multiple")
    refused(ops, lambda: att(q, k[:, :, :0], k[:, :, :0], 3), "multiple")
    refused(ops, lambda: att(torch.zeros(1, 1, 1, 257), torch.zeros(1, 1, 1, 257), torch.zeros(1, 1, 1, 257), 3), "dim must be")
    refused(ops, lambda: att(q, k, k, 0), "window")
    refused(ops, lambda: att(q, k, k, 3, -1), "sinks")
    refused(ops, lambda: att(q, k, k, 3, scale=float("nan")), "scale")
    refused(ops, lambda: att(q, k, k, 3, kv_lengths=torch.zeros(2)), "lengths must be INT32")
    refused(ops, lambda: att(q, k, k, 3, kv_lengths=torch.zeros(3, dtype=torch.int32)), "lengths must be [batch]")
    refused(ops, lambda: att(q, k, k, 3, q_lengths=torch.zeros(4, dtype=torch.int32)[::2]), "lengths must be [batch]")
    refused(ops, lambda: att(q, k, k, 3, out=q.half()), "out must have")
    refused(ops, lambda: att(q, k, k, 3, out=torch.zeros(1, 5, 4, 16).expand(2, 5, 4, 16)), "overlap")
    refused(ops, lambda: att(q, k, k, 3, lse=torch.zeros(2, 5, 4)), "lse must be")
    refused(ops, lambda: back(q, q, k, k, q, lse.half(), 3), "lse must be")
    refused(ops, lambda: back(q, q, k, k, q[:, :4], lse, 3), "gradOut, out and gradQ")
    refused(ops, lambda: back(q, q, k, k, q, lse, 3, grad_k=q), "gradK and gradV")
    refused(ops, lambda: back(q, q, k, k, q, lse, 3, grad_v=torch.zeros(1, 1, 1, 16).expand(2, 9, 2, 16)), "overlap")
    with pytest.raises(IndexError):
        att(q[0, 0], k, k, 3)


def test_tensors_without_data(ops):
    """A tensor with elements and no address is refused before a kernel could read it; an empty one needs none."""
    L = ops.lib()

    def tensor(*shape, dtype=ops.ACL_FLOAT, data=None):
        dims = (ctypes.c_int64 * len(shape))(*shape)
        return ctypes.c_void_p(L.aclCreateTensor(dims, len(shape), dtype, None, 0, ops.ACL_FORMAT_ND, dims, len(shape), data))

    n, e = ctypes.c_uint64(0), ctypes.c_void_p(None)
    some = ctypes.c_void_p(4096)
    for rows, status in ((3, NULLPTR), (0, 0)):
        x, y, bare = tensor(rows, 8, data=some), tensor(rows, 8, data=some), tensor(rows, 8)
        for args in ((x, None, None, y), (bare, None, None, y), (x, bare, None, y), (x, None, None, bare)):
            got = L.aclnnResidualRmsNormGetWorkspaceSize(args[0], args[1], args[2], 1e-6, args[3], None, None, ctypes.byref(n), ctypes.byref(e))
            assert got == (status if bare in args else 0)
            if got == 0:
                L.aclDestroyAclOpExecutor(e)
    q, k, bare = tensor(1, 2, 2, 8, data=some), tensor(1, 4, 1, 8, data=some), tensor(1, 4, 1, 8)
    got = L.aclnnWindowAttentionGetWorkspaceSize(q, k, bare, None, None, 3, 0, 1.0, q, None, ctypes.byref(n), ctypes.byref(e))
    assert got == NULLPTR
    got = L.aclnnRotaryEmbeddingGetWorkspaceSize(q, None, tensor(1, 2, dtype=ops.ACL_INT64), tensor(4, data=some), None, False, 1.0, q, None,
                                                 ctypes.byref(n), ctypes.byref(e))
    assert got == NULLPTR


@pytest.mark.parametrize("code", ["ACL_BF16", "ACL_FLOAT"])
@pytest.mark.parametrize("sinks", [0, 4, 1000, 2 ** 20, 2 ** 40])
def test_workspace_of_many_sinks(ops, code, sinks):
    """However many sinks there are, the sums of the blocks that share their queries stay small (the tensors take 4 GiB and more)."""
    L = ops.lib()

    def tensor(*shape, dtype):
        dims = (ctypes.c_int64 * len(shape))(*shape)
        return ctypes.c_void_p(L.aclCreateTensor(dims, len(shape), dtype, None, 0, ops.ACL_FORMAT_ND, dims, len(shape), ctypes.c_void_p(4096)))

    dtype, tokens, heads, kv, d = getattr(ops, code), 2 ** 20, 16, 4, 128
    q, k = tensor(1, tokens, heads, d, dtype=dtype), tensor(1, tokens, kv, d, dtype=dtype)
    lse = tensor(1, heads, tokens, dtype=ops.ACL_FLOAT)
    n, e = ctypes.c_uint64(0), ctypes.c_void_p(None)
    got = L.aclnnWindowAttentionBackwardGetWorkspaceSize(q, q, k, k, q, lse, None, None, 64, sinks, 0.1, q, k, k, ctypes.byref(n), ctypes.byref(e))
    assert got == 0 and n.value < 2 ** 30
    L.aclDestroyAclOpExecutor(e)


def test_tensors_of_two_devices(ops):
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="one device"):
        ops.residual_rms_norm(x, torch.zeros(2, 8, device="meta"))


def test_rotary_accepts_positions_that_broadcast(ops):
    q, f = torch.zeros(2, 3, 4, 2, 8), torch.zeros(4)
    for shape in ((2, 1, 1), (1, 3, 1), (1, 1, 4), (2, 1, 4), (2, 3, 1), (1, 3, 4), (3, 1), (1, 1, 1)):
        for t in (torch.int32, torch.int64):
            accepted(lambda: ops.rotary_embedding(q, None, torch.zeros(shape, dtype=t), f))


def test_rotary_positions_by_axes_broadcast(ops):
    q, f = torch.zeros(2, 5, 4, 16), torch.zeros(8)
    for shape in ((3, 5), (3, 1, 5), (3, 2, 1), (3, 1), (3,), (3, 2, 5)):
        accepted(lambda: ops.rotary_embedding(q, None, torch.zeros(shape, dtype=torch.int64), f, sections=(4, 2, 2)))
        accepted(lambda: ops.rotary_embedding_backward(q, None, torch.zeros(shape, dtype=torch.int32), f, sections=(4, 2, 2)))
        refused(ops, lambda: ops.rotary_embedding(q, None, torch.zeros(shape, dtype=torch.int64), f, sections=(4, 4)), "positions must be")
    accepted(lambda: ops.rotary_embedding(q[0, 0], None, torch.zeros(2, dtype=torch.int64), f, sections=(4, 4)))
    for shape in ((3, 4), (3, 5, 2), (3, 2, 2, 5)):
        with pytest.raises(RuntimeError, match="expand"):
            ops.rotary_embedding(q, None, torch.zeros(shape, dtype=torch.int64), f, sections=(4, 2, 2))
    refused(ops, lambda: ops.rotary_embedding(q, None, torch.tensor(3), f, sections=(8,)), "positions must be")


@pytest.mark.parametrize("code", ["ACL_BF16", "ACL_FLOAT"])
@pytest.mark.parametrize("batch,tokens,kv,group,sinks", [(64, 4096, 8, 1, 4), (64, 4096, 8, 4, 130), (256, 2048, 16, 1, 1), (16, 32768, 8, 1, 300)])
def test_workspace_of_many_sequences(ops, code, batch, tokens, kv, group, sinks):
    """However many sequences have sinks, the sums of the blocks that share their queries take less than the gradient of the keys."""
    L = ops.lib()

    def tensor(*shape, dtype):
        dims = (ctypes.c_int64 * len(shape))(*shape)
        return ctypes.c_void_p(L.aclCreateTensor(dims, len(shape), dtype, None, 0, ops.ACL_FORMAT_ND, dims, len(shape), ctypes.c_void_p(4096)))

    dtype, d, elem = getattr(ops, code), 128, 2 if code == "ACL_BF16" else 4
    q, k = tensor(batch, tokens, kv * group, d, dtype=dtype), tensor(batch, tokens, kv, d, dtype=dtype)
    lse = tensor(batch, kv * group, tokens, dtype=ops.ACL_FLOAT)
    n, e = ctypes.c_uint64(0), ctypes.c_void_p(None)
    got = L.aclnnWindowAttentionBackwardGetWorkspaceSize(q, q, k, k, q, lse, None, None, 64, sinks, 0.1, q, k, k, ctypes.byref(n), ctypes.byref(e))
    statistics = 2 * 4 * batch * kv * group * (tokens + 256)
    assert got == 0 and n.value - statistics < batch * tokens * kv * d * elem
    L.aclDestroyAclOpExecutor(e)


def test_scalars_beyond_fp32(ops):
    """Finite in 64 bits is not enough: the kernels take them in 32."""
    x, q, f, p = torch.zeros(2, 3, 8), torch.zeros(2, 5, 4, 16), torch.zeros(8), torch.arange(5)
    for big in (1e39, 1e300):
        refused(ops, lambda: ops.residual_rms_norm(x, eps=big), "eps")
        refused(ops, lambda: ops.residual_rms_norm_quant(x, eps=big), "eps")
        for sign in (1, -1):
            refused(ops, lambda: ops.rotary_embedding(q, None, p, f, scale=sign * big), "scale")
            refused(ops, lambda: ops.rotary_embedding_backward(q, None, p, f, scale=sign * big), "scale")
            refused(ops, lambda: ops.window_attention(q, q, q, 3, scale=sign * big), "scale")
            refused(ops, lambda: ops.window_attention_backward(q, q, q, q, q, torch.zeros(2, 4, 5), 3, scale=sign * big), "scale")
    accepted(lambda: ops.residual_rms_norm(x, eps=3e38))
    accepted(lambda: ops.rotary_embedding(q, None, p, f, scale=-3e38))
    accepted(lambda: ops.window_attention(q, q, q, 3, scale=3e38))


def test_attention_refuses_too_many_heads_to_a_key_head(ops):
    """Their products with 8 queries would not fit 32 bits."""
    L = ops.lib()

    def tensor(*shape):
        dims = (ctypes.c_int64 * len(shape))(*shape)
        return ctypes.c_void_p(L.aclCreateTensor(dims, len(shape), ops.ACL_FLOAT, None, 0, ops.ACL_FORMAT_ND, dims, len(shape), ctypes.c_void_p(4096)))

    n, e = ctypes.c_uint64(0), ctypes.c_void_p(None)
    for heads, status in ((2 ** 24, 0), (2 ** 24 + 1, INVALID), (2 ** 28, INVALID)):
        q, k, lse = tensor(1, 8, heads, 1), tensor(1, 8, 1, 1), tensor(1, heads, 8)
        got = L.aclnnWindowAttentionGetWorkspaceSize(q, k, k, None, None, 3, 0, 1.0, q, lse, ctypes.byref(n), ctypes.byref(e))
        assert got == status
        if got == 0:
            L.aclDestroyAclOpExecutor(e)
        assert L.aclnnWindowAttentionBackwardGetWorkspaceSize(q, q, k, k, q, lse, None, None, 3, 0, 1.0, q, k, k, ctypes.byref(n),
                                                              ctypes.byref(e)) == status
        if status == 0:
            L.aclDestroyAclOpExecutor(e)


def test_rotary_accepts_positions_by_axes_that_broadcast_between(ops):
    q, f = torch.zeros(2, 3, 4, 5, 2, 8), torch.zeros(4)
    for shape in ((1, 3, 1, 5), (2, 1, 4, 1), (1, 1, 4, 1), (1, 3, 4, 1), (2, 1, 1, 5)):
        accepted(lambda: ops.rotary_embedding(q, None, torch.zeros((2, *shape), dtype=torch.int64), f, sections=(3, 1)))
        accepted(lambda: ops.rotary_embedding(q, None, torch.zeros(shape, dtype=torch.int32), f))
