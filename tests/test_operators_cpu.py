"""Host-side checks of the operators around the grouped GEMM: every refusal comes before the device is touched, sizes of scratch
need no device.  No GPU."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P, I, L = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
BF16, F16, F8, F32 = 0, 1, 2, 4


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.path.join(ROOT, "grouped_gemm_amd", "libgrouped_gemm_hip.so"))
    lib.gg_last_error.restype = ctypes.c_char_p
    lib.gg_route.argtypes = [P, I, L, L, L, I, I] + [P] * 8
    lib.gg_route_backward.argtypes = [P, I, L, L, L, I, I] + [P] * 5
    lib.gg_moe_few_tokens.argtypes = [P] * 6 + [I, L, L, L, L, L, I, P, P]
    lib.gg_lora.argtypes = [P] * 7 + [I, L, L, L, L, L, P, P]
    for name, count in (("gg_route_scratch_bytes", 3), ("gg_lora_scratch_bytes", 5)):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [L] * count, ctypes.c_uint64
    lib.gg_moe_few_tokens_scratch_bytes.argtypes, lib.gg_moe_few_tokens_scratch_bytes.restype = [L] * 5 + [I], ctypes.c_uint64
    return lib


def test_route_argument_errors_need_no_device(lib):
    x = 4096   # (an address: refused before anything reads it)

    def call(logits=x, dtype=F32, tokens=100, experts=8, top_k=2, score=0, weights=x, chosen=x, sizes=x, row_index=x, order=x, scratch=x):
        return lib.gg_route(logits, dtype, tokens, experts, top_k, score, 1, weights, chosen, sizes, row_index, order, None, scratch, None)

    for kw, code, text in [(dict(dtype=F8), -1, b"dtype"), (dict(tokens=-1), -1, b"tokens"), (dict(experts=0), -1, b"experts"),
                           (dict(top_k=0), -1, b"top_k"), (dict(top_k=9), -1, b"top_k"), (dict(experts=1025), -2, b"at most"),
                           (dict(experts=64, top_k=33), -2, b"at most"), (dict(tokens=1 << 30, top_k=2), -2, b"2^31"),
                           (dict(score=2), -1, b"score"), (dict(logits=None), -1, b"logits"), (dict(weights=None), -1, b"null"),
                           (dict(sizes=None), -1, b"null"), (dict(order=None), -1, b"null"), (dict(scratch=None), -1, b"scratch")]:
        assert call(**kw) == code, kw
        assert text in lib.gg_last_error(), (kw, lib.gg_last_error())
    back = lambda **kw: lib.gg_route_backward(*[{**dict(logits=x, dtype=F32, tokens=4, experts=8, top_k=2, score=0, normalize=1, chosen=x, wg=x, mg=x, out=x,  # noqa: E731
                                                        stream=None), **kw}[k] for k in ("logits", "dtype", "tokens", "experts", "top_k", "score", "normalize",
                                                                                         "chosen", "wg", "mg", "out", "stream")])
    assert back(chosen=None) == -1 and back(out=None) == -1 and back(dtype=7) == -1
    assert back(tokens=0, logits=None, chosen=None, out=None) == 0   # nothing to do


def test_few_tokens_argument_errors_need_no_device(lib):
    x = 4096

    def call(a=x, dtype=BF16, tokens=2, experts=4, top_k=2, hidden=64, ffn=64, scratch=x, out=x):
        return lib.gg_moe_few_tokens(a, x, x, x, x, out, dtype, tokens, experts, top_k, hidden, ffn, 0, scratch, None)

    for kw, code, text in [(dict(dtype=F32), -1, b"dtype"), (dict(tokens=-1), -1, b"tokens"), (dict(hidden=0), -1, b"hidden"),
                           (dict(tokens=65), -2, b"at most"), (dict(experts=1025), -2, b"at most"), (dict(top_k=33), -2, b"at most"),
                           (dict(ffn=1 << 22), -2, b"2^22"), (dict(tokens=64, top_k=32, experts=1024, hidden=(1 << 22) - 1, ffn=(1 << 22) - 1), -2, b"too large"),
                           (dict(a=None), -1, b"null"), (dict(out=None), -1, b"null"), (dict(scratch=None), -1, b"null"), (dict(scratch=x + 16), -2, b"256")]:
        assert call(**kw) == code, kw
        assert text in lib.gg_last_error(), (kw, lib.gg_last_error())
    assert call(tokens=0, a=None) == 0


def test_lora_argument_errors_need_no_device(lib):
    x = 4096

    def call(a=x, dtype=BF16, rows=2, num=4, rank=8, hin=64, hout=64, out=x, scratch=x):
        return lib.gg_lora(x, a, x, x, None, None, out, dtype, rows, num, rank, hin, hout, scratch, None)

    for kw, code, text in [(dict(dtype=F32), -1, b"dtype"), (dict(rows=-1), -1, b"rows"), (dict(num=0), -1, b"adapters"), (dict(rank=0), -1, b"rank"),
                           (dict(rank=257), -2, b"rank"), (dict(rows=1 << 31), -2, b"2^31"), (dict(hin=1 << 22), -2, b"2^22"),
                           (dict(a=None), -1, b"null"), (dict(out=None), -1, b"null"), (dict(scratch=None), -1, b"null"), (dict(scratch=x + 8), -2, b"16")]:
        assert call(**kw) == code, kw
        assert text in lib.gg_last_error(), (kw, lib.gg_last_error())
    assert call(rows=0, a=None) == 0


def test_scratch_sizes_need_no_device(lib):
    assert lib.gg_route_scratch_bytes(1, 64, 6) == 0 and lib.gg_route_scratch_bytes(64, 64, 6) == 0
    # counts and mass of at most 512 workgroups
    assert 0 < lib.gg_route_scratch_bytes(65536, 256, 8) <= 2 * 256 * 512 * 4
    assert lib.gg_route_scratch_bytes(100, 0, 1) == 0 and lib.gg_route_scratch_bytes(100, 8, 33) == 0
    t, k, hidden, ffn = 3, 2, 100, 70
    # two rows of activations for each slot, and at least one of sums
    assert lib.gg_moe_few_tokens_scratch_bytes(t, 4, k, hidden, ffn, 0) >= t * k * (2 * ffn * 2 + hidden * 4)
    assert lib.gg_moe_few_tokens_scratch_bytes(65, 4, k, hidden, ffn, 0) == 0
    assert lib.gg_lora_scratch_bytes(10, 4, 16, 64, 64) >= 10 * 16 * 4
    assert lib.gg_lora_scratch_bytes(0, 4, 16, 64, 64) == 0 and lib.gg_lora_scratch_bytes(10, 4, 300, 64, 64) == 0


def test_cpu_tensors_are_refused():
    from grouped_gemm import ops
    x = torch.zeros(2, 16, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.route(x.float(), 2)
    experts, weights = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.moe_few_tokens(x, torch.zeros(3, 16, 8, dtype=x.dtype), torch.zeros(3, 4, 16, dtype=x.dtype), experts, weights)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.lora(x, torch.zeros(3, 4, 16, dtype=x.dtype), torch.zeros(3, 8, 4, dtype=x.dtype), torch.zeros(2, dtype=torch.int32))


def test_shapes_and_types_are_checked_before_the_device():
    from grouped_gemm import ops
    with pytest.raises(RuntimeError, match="score"):
        ops.route(torch.zeros(2, 8), 2, score="relu")
    with pytest.raises(RuntimeError, match="top_k"):
        ops.route(torch.zeros(2, 8), 0)
    x = torch.zeros(2, 16, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="even"):
        ops.moe_few_tokens(x, torch.zeros(3, 16, 7, dtype=x.dtype), torch.zeros(3, 4, 16, dtype=x.dtype), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2))
    with pytest.raises(RuntimeError, match="rank"):
        ops.lora(x, torch.zeros(3, 4, 16, dtype=x.dtype), torch.zeros(3, 8, 5, dtype=x.dtype), torch.zeros(2, dtype=torch.int32))
