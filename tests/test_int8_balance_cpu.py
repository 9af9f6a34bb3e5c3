"""Host-side checks of the products of 8-bit integers, the rows quantised for them and the balance loss: every refusal comes before the
device is touched, sizes of scratch need no device.  No GPU."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P, I, L = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
BF16, F16, F8, F32 = 0, 1, 2, 4


class Args(ctypes.Structure):
    _fields_ = [("struct_bytes", ctypes.c_uint32), ("dtype", ctypes.c_int32), ("a", P), ("b", P), ("c", P), ("batch_sizes", P),
                ("batch_sizes_on_device", ctypes.c_int32), ("trans_a", ctypes.c_int32), ("trans_b", ctypes.c_int32), ("accumulate_f32", ctypes.c_int32),
                ("num_groups", L), ("tokens", L), ("hidden_in", L), ("hidden_out", L), ("workspace", P), ("workspace_bytes", ctypes.c_uint64),
                ("flags", ctypes.c_int32), ("reserved0", ctypes.c_int32), ("stream", P), ("a_row_index", P), ("b_row_index", P), ("c_row_index", P),
                ("a_num_rows", L), ("c_num_rows", L), ("epilogue", ctypes.c_int32), ("b_num_rows", ctypes.c_int32), ("size_status", P)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.path.join(ROOT, "grouped_gemm_amd", "libgrouped_gemm_hip.so"))
    lib.gg_last_error.restype = ctypes.c_char_p
    lib.gg_quantize_rows.argtypes = [P, I, L, L, L, P, L, P, P, P]
    lib.gg_swiglu_quantize.argtypes = [P, I, L, L, L, P, P, P]
    lib.gg_gmm_int8.argtypes = [P, P, P]
    lib.gg_gmm_int8_workspace_bytes.argtypes, lib.gg_gmm_int8_workspace_bytes.restype = [P], ctypes.c_uint64
    lib.gg_balance.argtypes = [P, I, L, L, L, I, P, P, L] + [P] * 8
    lib.gg_balance_backward.argtypes = [P, I, L, L, I, P, L] + [P] * 7
    lib.gg_balance_scratch_bytes.argtypes, lib.gg_balance_scratch_bytes.restype = [L] * 4, ctypes.c_uint64
    return lib


def _refuses(lib, call, cases):
    for kw, code, text in cases:
        assert call(**kw) == code, kw
        assert text in lib.gg_last_error(), (kw, lib.gg_last_error())


def test_quantize_argument_errors_need_no_device(lib):
    x = 4096   # (an address: refused before anything reads it)

    def rows(src=x, dtype=BF16, rows=4, cols=64, stride=64, index=None, x_rows=4, q=x, scales=x):
        return lib.gg_quantize_rows(src, dtype, rows, cols, stride, index, x_rows, q, scales, None)

    _refuses(lib, rows, [(dict(dtype=F8), -1, b"dtype"), (dict(rows=-1), -1, b"rows"), (dict(cols=0), -1, b"cols"), (dict(cols=1 << 22), -2, b"2^22"),
                         (dict(stride=63), -1, b"overlap"), (dict(x_rows=3), -1, b"x_rows"), (dict(x_rows=-1, index=x), -1, b"x_rows"),
                         (dict(q=None), -1, b"null"), (dict(scales=None), -1, b"null"), (dict(src=None), -1, b"null"), (dict(rows=1 << 40, x_rows=1 << 40), -2, b"2^40")])
    assert rows(rows=0, src=None, q=None, scales=None) == 0

    def gated(src=x, dtype=BF16, rows=4, cols=64, stride=128, q=x, scales=x):
        return lib.gg_swiglu_quantize(src, dtype, rows, cols, stride, q, scales, None)

    _refuses(lib, gated, [(dict(dtype=F8), -1, b"dtype"), (dict(rows=-1), -1, b"rows"), (dict(stride=127), -1, b"overlap"), (dict(src=None), -1, b"null"),
                          (dict(q=None), -1, b"null"), (dict(cols=0), -1, b"cols")])
    assert gated(rows=0, src=None) == 0


def _args(sizes=(3, 4), **kw):
    host = (ctypes.c_int64 * len(sizes))(*sizes)
    a = Args(struct_bytes=ctypes.sizeof(Args), dtype=BF16, trans_b=1, a=4096, b=8192, c=16384, batch_sizes=ctypes.cast(host, P), num_groups=len(sizes), tokens=7,
             hidden_in=64, hidden_out=32)
    for k, v in kw.items():
        setattr(a, k, v)
    return a, host


def test_gmm_int8_argument_errors_need_no_device(lib):
    def call(a_scales=4096, b_scales=4096, **kw):
        args, host = _args(**kw)
        return lib.gg_gmm_int8(ctypes.byref(args), a_scales, b_scales)

    _refuses(lib, call, [(dict(struct_bytes=8), -1, b"struct_bytes"), (dict(dtype=F8), -1, b"dtype"), (dict(dtype=F32), -1, b"dtype"), (dict(trans_b=0), -1, b"trans"),
                         (dict(trans_a=1), -1, b"trans"), (dict(trans_a=1, trans_b=0), -1, b"trans"), (dict(epilogue=1), -1, b"epilogue"),
                         (dict(accumulate_f32=1), -1, b"epilogue"), (dict(a_row_index=4096), -1, b"indices"), (dict(c_row_index=4096), -1, b"indices"),
                         (dict(hidden_in=131072), -2, b"131071"), (dict(hidden_out=1 << 22), -2, b"2^22"), (dict(tokens=1 << 31), -2, b"2^31"), (dict(tokens=-1), -1, b"negative"),
                         (dict(a=None), -1, b"null"), (dict(b=None), -1, b"null"), (dict(c=None), -1, b"null"), (dict(a_scales=None), -1, b"null"),
                         (dict(b_scales=None), -1, b"null"), (dict(batch_sizes=None), -1, b"batch_sizes"), (dict(c=16385), -2, b"aligned"),
                         (dict(a_scales=4098), -2, b"aligned"), (dict(b_scales=4097), -2, b"aligned")])
    assert lib.gg_gmm_int8(None, 4096, 4096) == -1
    assert call(tokens=0, a=None, b=None, c=None, a_scales=None, b_scales=None) == 0
    assert call(hidden_out=0, c=None) == 0 and call(num_groups=0, batch_sizes=None) == 0


def test_gmm_int8_limits_are_those_of_the_kernel_that_runs(lib):
    """More windows of rows and strips of columns than one launch of the kernel for few rows takes: refused where that kernel would run, not where the
    streaming one does (which then gets as far as the sizes, wrong here on purpose)."""
    def call(**kw):
        args, host = _args(sizes=(-1,) * kw.pop("groups"), **kw)
        return lib.gg_gmm_int8(ctypes.byref(args), 4096, 4096), lib.gg_last_error()

    for kw in (dict(groups=8, tokens=1 << 20, hidden_in=16, hidden_out=65536), dict(groups=512, tokens=4097, hidden_in=16, hidden_out=1 << 21)):
        rc, text = call(**kw)
        assert rc == -1 and b"negative" in text, (kw, rc, text)
        for odd in (dict(hidden_in=15), dict(a=4097), dict(b=8200)):
            rc, text = call(**{**kw, **odd})
            assert rc == -2 and b"too large" in text, (kw, odd, rc, text)
    rc, text = call(groups=512, tokens=4096, hidden_in=16, hidden_out=1 << 21)   # (few rows to a group)
    assert rc == -2 and b"too large" in text
    rc, text = call(groups=8, tokens=1 << 10, hidden_in=15, hidden_out=65536)
    assert rc == -1 and b"negative" in text


def test_gmm_int8_workspace_goes_by_the_sizes(lib):
    def wanted(sizes, hidden_in, hidden_out, tokens=None):
        args, host = _args(sizes=sizes, tokens=sum(sizes) if tokens is None else tokens, hidden_in=hidden_in, hidden_out=hidden_out)
        return lib.gg_gmm_int8_workspace_bytes(ctypes.byref(args))

    assert wanted([1, 1], 14336, 4096) > 0            # two strips of columns to a compute unit, a deep product
    assert wanted([1, 1], 256, 4096) == 0             # nothing to cut
    assert wanted([512] * 128, 7168, 4096) == 0       # more tiles than compute units
    assert wanted([300], 16384, 128) > 0              # a few deep tiles
    assert wanted([300], 16384, 121) > 0 and wanted([300], 16383, 128) > 0   # ... of any width; few windows of the kernel for any sizes
    assert wanted([3000], 16383, 4096) == 0           # (more of those than compute units)
    assert wanted([0, 0], 64, 64) == 0 and wanted([1], 0, 64) == 0
    assert lib.gg_gmm_int8_workspace_bytes(None) == 0


def test_balance_argument_errors_need_no_device(lib):
    x = 4096

    def call(logits=x, dtype=F32, tokens=100, experts=8, top_k=2, score=0, chosen=x, offsets=x, sequences=3, balance=x, z=x, counts=x, share=x, inverse=x, scratch=x):
        return lib.gg_balance(logits, dtype, tokens, experts, top_k, score, chosen, offsets, sequences, None, balance, z, counts, share, inverse, scratch, None)

    _refuses(lib, call, [(dict(dtype=F8), -1, b"dtype"), (dict(tokens=-1), -1, b"tokens"), (dict(experts=0), -1, b"experts"), (dict(top_k=9), -1, b"top_k"),
                         (dict(experts=1025), -2, b"at most"), (dict(experts=64, top_k=33), -2, b"at most"), (dict(tokens=1 << 30), -2, b"2^31"),
                         (dict(score=2), -1, b"score"), (dict(sequences=-1), -1, b"sequences"), (dict(sequences=2, offsets=None), -1, b"sequences"),
                         (dict(sequences=(1 << 31) - 1), -2, b"sequences"), (dict(logits=None), -1, b"logits"), (dict(chosen=None), -1, b"chosen"),
                         (dict(balance=None), -1, b"null"), (dict(z=None), -1, b"null"), (dict(counts=None), -1, b"null"), (dict(share=None), -1, b"null"),
                         (dict(inverse=None), -1, b"null"), (dict(scratch=None), -1, b"null")])

    def back(logits=x, dtype=F32, tokens=100, experts=8, score=0, offsets=x, sequences=3, share=x, inverse=x, out=x):
        return lib.gg_balance_backward(logits, dtype, tokens, experts, score, offsets, sequences, None, share, inverse, x, x, out, None)

    _refuses(lib, back, [(dict(dtype=F8), -1, b"dtype"), (dict(score=5), -1, b"score"), (dict(out=None), -1, b"null"), (dict(share=None), -1, b"null"),
                         (dict(inverse=None), -1, b"null"), (dict(logits=None), -1, b"logits"), (dict(offsets=None), -1, b"sequences")])
    assert back(tokens=0, logits=None, out=None) == 0


def test_balance_scratch_holds_a_row_for_every_unit(lib):
    bytes_for = lib.gg_balance_scratch_bytes
    assert bytes_for(1, 8, 2, 1) >= 2 * 8 * 8
    # at most 1024 workgroups and a row for each sequence, of masses and counts
    assert 1024 * 256 * 8 <= bytes_for(65536, 256, 8, 64) <= (1024 + 64 + 1) * (256 * 8 + 8) + 64 * 4 * 8 + 1024
    assert bytes_for(100, 0, 1, 1) == 0 and bytes_for(100, 8, 33, 1) == 0 and bytes_for(-1, 8, 2, 1) == 0 and bytes_for(100, 8, 2, -1) == 0
    assert bytes_for(0, 8, 2, 0) > 0


def test_cpu_tensors_are_refused():
    from grouped_gemm import ops
    with pytest.raises(RuntimeError, match="GPU"):
        ops.quantize_rows(torch.zeros(2, 16))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.swiglu_quantize(torch.zeros(2, 16))
    a, b = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(3, 8, 16, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.gmm_int8(a, torch.zeros(2), b, torch.zeros(3, 8), torch.tensor([1, 0, 1]))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.balance_loss(torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32))


def test_shapes_and_types_are_checked_before_the_device():
    from grouped_gemm import ops
    for x in (torch.zeros(2, 16, dtype=torch.float64), torch.zeros(2, 16, dtype=torch.int8)):
        with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
            ops.quantize_rows(x)
    for x in (torch.zeros(2, 0), torch.zeros(())):
        with pytest.raises(RuntimeError, match="at least one"):
            ops.quantize_rows(x)
    for x in (torch.zeros(4, 16).t(), torch.zeros(1, 16).expand(4, 16), torch.zeros(3, 4, 16).transpose(0, 1), torch.zeros(4, 32)[:, ::2]):
        with pytest.raises(RuntimeError, match="contiguous"):
            ops.quantize_rows(x)
    a, b, sizes = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(3, 8, 16, dtype=torch.int8), torch.tensor([1, 0, 1])
    good = dict(a=a, a_scales=torch.zeros(2), b=b, b_scales=torch.zeros(3, 8), batch_sizes=sizes)
    for kw, text in [(dict(a=a.float()), "int8"), (dict(a=a[0]), "int8"), (dict(b=b[0]), "int8"), (dict(b=b.short()), "int8"), (dict(a=a[:, :8]), "contraction"),
                     (dict(a_scales=torch.zeros(3)), "a_scales"), (dict(a_scales=torch.zeros(2).double()), "a_scales"), (dict(b_scales=torch.zeros(3, 7)), "b_scales"),
                     (dict(b_scales=torch.zeros(24)), "b_scales"), (dict(batch_sizes=sizes[:2]), "batch_sizes"), (dict(batch_sizes=sizes.int()), "batch_sizes"),
                     (dict(c=torch.zeros(2, 8)), "c must"), (dict(c=torch.zeros(2, 9, dtype=torch.bfloat16)), "c must"),
                     (dict(c=torch.zeros(2, 8, dtype=torch.bfloat16), dtype=torch.float16), "c must"), (dict(b=b.transpose(0, 1).contiguous().transpose(0, 1)), "contiguous")]:
        with pytest.raises(RuntimeError, match=text):
            ops.gmm_int8(**{**good, **kw})
    with pytest.raises(ValueError, match="dtype"):
        ops.gmm_int8(**good, dtype=torch.float32)
    logits, experts = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for args, kw, text in [((logits, experts.long()), {}, "experts"), ((logits, experts[:3]), {}, "experts"), ((logits.double(), experts), {}, "logits"),
                           ((logits[0], experts), {}, "2-d"), ((logits, experts), dict(score="relu"), "score"), ((logits, experts[:, :0]), {}, "top_k"),
                           ((logits, torch.zeros(4, 9, dtype=torch.int32)), {}, "top_k"), ((torch.zeros(8, 4).t(), experts), {}, "contiguous")]:
        with pytest.raises(RuntimeError, match=text):
            ops.balance_loss(*args, **kw)
