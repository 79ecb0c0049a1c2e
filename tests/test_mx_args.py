"""Arguments that the MX entry points refuse, checked before any device is
looked for: no GPU needed, nothing is launched (the buffers wrap made-up
addresses that are never touched)."""

from __future__ import annotations

import pytest

from qw3_b200 import build, ds3

FP8, FP4 = ds3.MXFP8, ds3.MXFP4
F32, F16, Q80 = ds3.TYPE_F32, ds3.TYPE_F16, ds3.TYPE_Q8_0


@pytest.fixture(scope="module", autouse=True)
def library():
    build.build()
    ds3.lib()


class Arena:
    """Distinct made-up buffers: each wraps its own 1 GiB of address space."""

    def __init__(self):
        self.next = 1 << 40

    def __call__(self, nbytes, shift=0):
        p = self.next + shift
        self.next += 1 << 30
        return ds3.buffer_wrap(p, nbytes)


@pytest.fixture
def buf():
    return Arena()


def refused(rc, word):
    assert rc == -1
    assert word in ds3.last_error(), ds3.last_error()


def quantize(buf, **k):
    a = dict(src=buf(4 * 4096), src_type=F32, q=buf(4096), scales=buf(128), to=FP8, n_rows=4, n_cols=1024)
    a.update(k)
    return ds3.mx_quantize(*a.values())


@pytest.mark.parametrize("change,word", [
    (dict(n_cols=1000), "32-element blocks"),
    (dict(n_cols=0), "32-element blocks"),
    (dict(to=2), "type 2"),
    (dict(src_type=Q80), "src_type"),
    (dict(n_rows=5), "holds"),
    (dict(n_rows=1 << 60), "too many"),
    (dict(src=None), "NULL"),
])
def test_quantize_refusals(buf, change, word):
    refused(quantize(buf, **change), word)


def test_quantize_refuses_alignment_and_overlap(buf):
    refused(quantize(buf, src=buf(4 * 4096, 4)), "16-byte aligned")
    refused(quantize(buf, q=buf(4096, 8)), "16-byte aligned")
    src = buf(4 * 4096)
    refused(quantize(buf, src=src, q=ds3.buffer_view(src, 16, 4096)), "overlaps")
    q = buf(8192)
    refused(quantize(buf, q=q, scales=ds3.buffer_view(q, 4000, 128)), "overlaps")


@pytest.mark.parametrize("change,word", [
    (dict(n_cols=48), "32-element blocks"), (dict(from_=7), "type 7"), (dict(dst=None), "NULL"), (dict(n_rows=5), "holds"),
])
def test_dequantize_refusals(buf, change, word):
    a = dict(q=buf(4096), scales=buf(128), from_=FP8, dst=buf(4 * 4096), n_rows=4, n_cols=1024)
    a.update(change)
    refused(ds3.mx_dequantize(*a.values()), word)


def norm(buf, **k):
    rb = 4 * 64 * 4
    a = dict(x=buf(rb), residual=buf(rb), weight=buf(256), sum_out=buf(rb), norm_out=buf(rb), q=buf(256), scales=buf(8),
             n=64, n_rows=4, eps=1e-6)
    a.update(k)
    return ds3.add_rms_norm_mx(*a.values())


@pytest.mark.parametrize("change,word", [
    (dict(n=63), "32-element blocks"),
    (dict(n=16416), "16384"),
    (dict(n_rows=5), "holds"),
    (dict(x=None), "NULL"),
    (dict(weight=None), "NULL"),
    (dict(q=None), "NULL"),
])
def test_norm_refusals(buf, change, word):
    refused(norm(buf, **change), word)


def test_norm_refuses_partial_overlap(buf):
    x = buf(8192)
    refused(norm(buf, x=ds3.buffer_view(x, 0, 1024), sum_out=ds3.buffer_view(x, 16, 1024)), "overlaps")
    s = buf(1024)
    refused(norm(buf, sum_out=s, norm_out=s), "overlaps")
    refused(norm(buf, x=buf(1024, 4)), "16-byte aligned")
    r = buf(1024)
    refused(norm(buf, residual=r, norm_out=r), "overlaps")


@pytest.mark.parametrize("change,word", [
    (dict(n_expert=0), "n_expert"), (dict(n_expert=257), "n_expert"), (dict(n_used=0), "n_used"),
    (dict(n_tokens=1 << 30, n_used=2), "2^30"), (dict(n_tokens=5), "holds"), (dict(entries=None), "NULL"),
    (dict(offsets="idx"), "overlaps"),
])
def test_expert_rows_refusals(buf, change, word):
    a = dict(idx=buf(4 * 8 * 4), offsets=buf(65 * 4), entries=buf(4 * 8 * 4), row_of=buf(4 * 8 * 4), n_tokens=4,
             n_expert=64, n_used=8)
    a.update(change)
    if a["offsets"] == "idx":
        a["n_expert"] = 16
        a["offsets"] = a["idx"]
    refused(ds3.moe_expert_rows(*a.values()), word)


@pytest.mark.parametrize("which", ["idx", "offsets", "entries", "row_of"])
def test_expert_rows_refuses_odd_addresses(buf, which):
    a = dict(idx=buf(128), offsets=buf(65 * 4), entries=buf(128), row_of=buf(128), n_tokens=4, n_expert=64, n_used=8)
    a[which] = buf(65 * 4, 2)
    refused(ds3.moe_expert_rows(*a.values()), "4-byte aligned")


def matmul(buf, **k):
    # 4 experts, 8 rows, 256 -> 96
    a = dict(x_q=buf(8 * 256), x_scales=buf(64), x_rows=buf(32), x_div=1, offsets=buf(20), w_q=buf(4 * 96 * 256),
             w_scales=buf(4 * 96 * 8), w_type=FP8, out=buf(8 * 96 * 4), out_type=F32, out_rows=None, n_x=8, n_rows=8,
             n_expert=4, n_in=256, n_out=96)
    a.update(k)
    return ds3.moe_mx_matmul(*a.values())


@pytest.mark.parametrize("change,word", [
    (dict(w_type=5), "type 5"),
    (dict(n_expert=0), "n_expert"),
    (dict(n_expert=257), "n_expert"),
    (dict(x_div=0), "x_div"),
    (dict(n_in=0), "n_in"),
    (dict(n_in=250), "n_in"),
    (dict(n_in=160, w_type=FP4), "128"),
    (dict(n_out=0), "n_out"),
    (dict(out_type=Q80), "out_type"),
    (dict(n_rows=9, x_rows=None, n_x=8), "holds"),
    (dict(n_rows=9), "holds"),
    (dict(n_x=9), "holds"),
    (dict(offsets=None), "NULL"),
    (dict(w_scales=None), "NULL"),
    (dict(n_x=1 << 31), "2^31"),
    (dict(n_x=1 << 20, x_div=1 << 20), "2^31"),
])
def test_matmul_refusals(buf, change, word):
    refused(matmul(buf, **change), word)


def test_matmul_refuses_short_x_alignment_and_overlap(buf):
    refused(matmul(buf, x_rows=None, n_x=7), "without x_rows")
    refused(matmul(buf, x_q=buf(2048, 8)), "16-byte aligned")
    refused(matmul(buf, w_type=FP4, w_q=buf(4 * 96 * 256, 16)), "32-byte aligned")
    refused(matmul(buf, out=buf(8 * 96 * 4, 2)), "4-byte aligned")
    x = buf(8 * 256 + 8 * 96 * 4)
    refused(matmul(buf, x_q=x, out=ds3.buffer_view(x, 1024, 8 * 96 * 4)), "overlaps")


def swiglu(buf, **k):
    a = dict(x_q=buf(8 * 256), x_scales=buf(64), x_rows=buf(64), x_div=2, offsets=buf(20), gate_q=buf(4 * 96 * 256),
             gate_scales=buf(4 * 96 * 8), up_q=buf(4 * 96 * 256), up_scales=buf(4 * 96 * 8), w_type=FP8, row_weight=buf(64),
             act_q=buf(16 * 96), act_scales=buf(16 * 3), n_x=8, n_rows=16, n_expert=4, n_in=256, n_ff=96)
    a.update(k)
    return ds3.moe_mx_swiglu(*a.values())


@pytest.mark.parametrize("change,word", [
    (dict(n_ff=80), "n_ff"),
    (dict(up_q=None), "NULL"),
    (dict(up_scales=None), "NULL"),
    (dict(act_scales=None), "NULL"),
    (dict(x_div=3), "row_weight"),
    (dict(n_rows=17), "holds"),
])
def test_swiglu_refusals(buf, change, word):
    refused(swiglu(buf, **change), word)


def test_swiglu_refuses_unaligned_rows(buf):
    refused(swiglu(buf, act_q=buf(16 * 96, 4)), "16-byte aligned")


def test_good_arguments_reach_the_device_check(buf):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present: these addresses must not be launched on")
    for rc in (quantize(buf), norm(buf), matmul(buf), swiglu(buf)):
        refused(rc, "not initialised")


def many_rows(op, mapped, n):
    """n rows of 32 elements, with buffers that would hold them."""
    at = iter(range(1 << 43, 1 << 47, 1 << 43))
    huge = lambda: ds3.buffer_wrap(next(at), 1 << 42)  # noqa: E731
    a = dict(x_q=huge(), x_scales=huge(), x_rows=huge() if mapped else None, x_div=1, n_x=n, n_rows=n, n_expert=1, n_in=32)
    a.update(dict(out=huge(), out_type=F16, n_out=1) if op is matmul else
             dict(act_q=huge(), act_scales=huge(), row_weight=None, n_ff=32))
    return op(Arena(), **a)


@pytest.mark.parametrize("n", [(1 << 30) + 1, (1 << 31) - 223, (1 << 31) - 1])
@pytest.mark.parametrize("mapped", [False, True])
@pytest.mark.parametrize("op", [matmul, swiglu])
def test_products_refuse_more_than_2_30_rows(op, mapped, n):
    """Near 2^31 the kernels' counts of row blocks would leave 31 bits."""
    refused(many_rows(op, mapped, n), "2^30")


@pytest.mark.parametrize("mapped", [False, True])
@pytest.mark.parametrize("op", [matmul, swiglu])
def test_products_take_2_30_rows(op, mapped):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present: these addresses must not be launched on")
    refused(many_rows(op, mapped, 1 << 30), "not initialised")
