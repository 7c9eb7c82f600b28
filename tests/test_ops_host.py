"""CPU checks of the device-buffer operators: every entry point of include/czg_ops.h is
exported, and calls that the host can see to be wrong are refused before any device work
(these calls reach no GPU: nothing is queued for them)."""
import ctypes as C
import os
import re

import pytest
import torch

OK, E_ARG, E_UNSUPPORTED, E_LIMIT = 0, 1, 3, 9
F32, BF16, F16 = 0, 1, 2
P = 4096      # a pointer that is aligned and never followed


@pytest.fixture(scope="module")
def ops():
    from compress_zip_b200 import build, ops

    build.build()
    return ops


def test_library_exports_header_symbols(root, ops):
    hdr = open(os.path.join(root, "include", "czg_ops.h")).read()
    hdr = re.sub(r"/\*.*?\*/", "", hdr, flags=re.S)
    declared = set(re.findall(r"\b(czg_[a-z0-9_]+)\s*\(", hdr))
    assert declared == set(ops.EXPORTS)
    for name in declared:
        assert hasattr(ops.lib(), name)


def refused(ops, want, text, fn, *args):
    got = getattr(ops.lib(), fn)(*args)
    assert got == want, (got, ops.lib().czg_ops_last_error())
    if want != OK:
        assert text in ops.lib().czg_ops_last_error().decode()


@pytest.mark.parametrize("want,text,args", [
    (OK, "", (P, BF16, 8, 0, 8, P, 16, P, None)),
    (E_ARG, "negative", (P, BF16, 8, -1, 8, P, 16, P, None)),
    (E_ARG, "at least 1", (P, BF16, 8, 2, 0, P, 16, P, None)),
    (E_LIMIT, "2^31", (P, BF16, 8, 1 << 31, 8, P, 16, P, None)),
    (E_ARG, "null", (None, BF16, 8, 2, 8, P, 16, P, None)),
    (E_ARG, "null", (P, BF16, 8, 2, 8, None, 16, P, None)),
    (E_ARG, "null", (P, BF16, 8, 2, 8, P, 16, None, None)),
    (E_ARG, "dtype", (P, 3, 8, 2, 8, P, 16, P, None)),
    (E_ARG, "aligned", (P + 1, BF16, 8, 2, 8, P, 16, P, None)),
    (E_ARG, "16-byte", (P, BF16, 8, 2, 8, P + 8, 16, P, None)),
    (E_ARG, "16-byte", (P, BF16, 8, 2, 8, P, 24, P, None)),
    (E_ARG, "overlap", (P, BF16, 17, 2, 17, P, 16, P, None)),
])
def test_quantize_refusals(ops, want, text, args):
    refused(ops, want, text, "czg_quantize_rows", *args)


def linear_args(**over):
    a = dict(x=P, ldx=64, xs=P, w=P, ldw=64, ws=P, bias=None, m=2, n=3, k=50, out=1 << 20, kind=BF16, ldo=3, stream=None)
    a.update(over)
    return tuple(a.values())


@pytest.mark.parametrize("want,text,over", [
    (OK, "", dict(m=0)), (OK, "", dict(n=0)),
    (E_ARG, "negative", dict(m=-1)), (E_ARG, "at least 1", dict(k=0)),
    (E_LIMIT, "MAX_K", dict(k=131072, ldx=131072, ldw=131072)), (E_LIMIT, "2^31", dict(n=1 << 31)),
    (E_ARG, "null", dict(x=None)), (E_ARG, "null", dict(xs=None)), (E_ARG, "null", dict(w=None)),
    (E_ARG, "null", dict(ws=None)), (E_ARG, "null", dict(out=None)), (E_ARG, "out_dtype", dict(kind=-1)),
    (E_ARG, "16-byte", dict(ldx=50)), (E_ARG, "16-byte", dict(w=P + 4)), (E_ARG, "overlap", dict(ldw=48)),
    (E_ARG, "aligned", dict(out=P + 2, kind=F32)), (E_ARG, "overlap", dict(ldo=2)),
    (E_ARG, "over x", dict(out=P)), (E_ARG, "over x", dict(out=P + 64)), (E_ARG, "over w", dict(x=P + 4096, out=P + 128)),
    (E_ARG, "over x", dict(out=P + 48, ldo=32)), (E_ARG, "over w", dict(x=1 << 21, w=P, ldw=4096, out=P + 4096)),
])
def test_linear_refusals(ops, want, text, over):
    refused(ops, want, text, "czg_linear_i8", *linear_args(**over))


def test_linear_dynamic_refusals(ops):
    L = ops.lib()
    need = L.czg_linear_i8_workspace(21, 50)
    assert need == 21 * 64 + 96 and L.czg_linear_i8_workspace(0, 50) == 0
    assert L.czg_linear_i8_workspace(2, 50) == 0      # a few short rows take none

    def call(ws=P, n_ws=need, x=P, kind=BF16):
        return L.czg_linear_i8_dynamic(x, kind, 50, P, 64, P, None, 21, 3, 50, 1 << 20, BF16, 3, ws, n_ws, None)

    for args, text in ((dict(ws=None), "workspace"), (dict(ws=P + 8), "workspace"), (dict(n_ws=need - 1), "too small"),
                       (dict(x=None), "null"), (dict(kind=9), "dtype")):
        assert call(**args) == E_ARG and text in L.czg_ops_last_error().decode()


def cache(ops, **over):
    a = dict(k=P, v=P, scales=P, weights=P, status=P, n_slots=4, n_heads=2, capacity=100, head_dim=64)
    a.update(over)
    return C.byref(ops._KV4(*a.values()))


@pytest.mark.parametrize("want,text,over", [
    (E_ARG, "null", dict(k=None)), (E_ARG, "null", dict(scales=None)), (E_ARG, "null", dict(status=None)),
    (E_ARG, "at least one", dict(n_slots=0)), (E_ARG, "at least one", dict(capacity=-1)),
    (E_ARG, "aligned", dict(v=P + 8)), (E_ARG, "aligned", dict(scales=P + 4)), (E_UNSUPPORTED, "head_dim", dict(head_dim=96)),
])
def test_cache_refusals(ops, want, text, over):
    c = cache(ops, **over)
    refused(ops, want, text, "czg_kv4_append", c, P, 1, 1, 1, P, 1, 1, 1, BF16, P, P, 2, 1, None)
    refused(ops, want, text, "czg_kv4_read", c, P, P, 2, 1, P, P, BF16, None)
    refused(ops, want, text, "czg_kv4_attend", c, P, 256, 256, 64, BF16, P, P, 2, 1, 4, 100, 0.1, P, 256, 256, 64, P, 1 << 40, None)
    refused(ops, want, text, "czg_kv4_evict", c, P, P, 2, 100, 10, 2, P, P + 64, None)


def test_kv4_call_refusals(ops):
    c = cache(ops)

    def append(k=P, v=P, kind=BF16, slots=P, lengths=P, b=2, t=1):
        return ("czg_kv4_append", c, k, 1, 1, 1, v, 1, 1, 1, kind, slots, lengths, b, t, None)

    def attend(q=P, kind=BF16, slots=P, b=2, t=1, hq=4, max_len=100, out=1 << 20, ws=P, n_ws=1 << 40, os=(256, 256, 64)):
        return ("czg_kv4_attend", c, q, 256, 256, 64, kind, slots, P, b, t, hq, max_len, 0.1, out, *os, ws, n_ws, None)

    def evict(c=c, lengths=P, b=2, max_len=100, budget=10, recent=2, new=P + 64):
        return ("czg_kv4_evict", c, P, lengths, b, max_len, budget, recent, P, new, None)

    for want, text, call in (
            (OK, "", append(b=0)), (OK, "", append(t=0)), (E_ARG, "negative", append(b=-1)), (E_ARG, "null", append(k=None)),
            (E_ARG, "null", append(slots=None)), (E_ARG, "dtype", append(kind=7)), (E_ARG, "aligned", append(v=P + 1)),
            (E_LIMIT, "65,535", append(b=65536)),
            (OK, "", attend(b=0)), (OK, "", attend(t=0)), (E_ARG, "multiple", attend(hq=3)), (E_ARG, "multiple", attend(hq=0)),
            (E_UNSUPPORTED, "bf16 or fp16", attend(kind=F32)), (E_ARG, "null", attend(q=None)), (E_ARG, "null", attend(out=None)),
            (E_ARG, "negative", attend(max_len=-1)), (E_ARG, "workspace", attend(ws=P + 8)),
            (E_ARG, "overlap", attend(os=(0, 256, 64))), (E_ARG, "over q", attend(out=P + 128)), (E_ARG, "over q", attend(out=P - 64)),
            (E_ARG, "over q", attend(out=P, os=(512, 256, 64))), (E_ARG, "workspace", attend(out=P, ws=P + 8)),
            (OK, "", evict(b=0)), (E_ARG, "budget", evict(budget=0)), (E_ARG, "budget", evict(recent=11)),
            (E_ARG, "budget", evict(recent=-1)), (E_ARG, "weights", evict(c=cache(ops, weights=None))),
            (E_LIMIT, "EVICT_MAX", evict(max_len=(1 << 20) + 1)), (E_ARG, "new_lengths", evict(new=P)),
            (E_ARG, "null", evict(lengths=None)), (E_LIMIT, "65,534", evict(b=65535)),
            (OK, "", ("czg_kv4_read", c, P, P, 2, 0, P, P, BF16, None)),
            (OK, "", ("czg_kv4_read", c, P, P, 2, 3, None, None, BF16, None)),
            (E_ARG, "16-byte", ("czg_kv4_read", c, P, P, 2, 3, P + 8, P, BF16, None)),
            (E_ARG, "negative", ("czg_kv4_read", c, P, P, 2, -1, P, P, BF16, None))):
        refused(ops, want, text, *call)


def test_python_refusals(ops):
    x = torch.zeros(4, 32)
    q = ops.QRows(torch.zeros(8, 32, dtype=torch.int8), torch.ones(8))
    for text, call in (
            ("float32, bfloat16", lambda: ops.quantize_rows(x.double())),
            ("2-D", lambda: ops.quantize_rows(x.t())),
            ("CUDA device", lambda: ops.quantize_rows(x)),
            ("rows of 30", lambda: ops.linear_i8(x[:, :30], q)),
            ("out_dtype", lambda: ops.linear_i8(x, q, out_dtype=torch.int8)),
            ("shape", lambda: ops.linear_i8(x, q, out=torch.zeros(4, 9))),
            ("out_dtype", lambda: ops.linear_i8(x, q, out=torch.zeros(4, 8), out_dtype=torch.float16)),
            ("bias", lambda: ops.linear_i8(x, q, bias=torch.zeros(7))),
            ("bias", lambda: ops.linear_i8(x, q, bias=torch.zeros(8, dtype=torch.float16))),
            ("CUDA device", lambda: ops.linear_i8(x, q)),
            ("one scale a row", lambda: ops.linear_i8(x, ops.QRows(q.codes, torch.ones(7)))),
            ("16-byte", lambda: ops.linear_i8(x[:, :24], ops.QRows(q.codes[:, 1:25], q.scales))),
            ("int8", lambda: ops.linear_i8(x, ops.QRows(q.codes.float(), q.scales)))):
        with pytest.raises(ValueError, match=text):
            call()
    k = torch.zeros(2, 1, 16, 32, dtype=torch.uint8)
    s = torch.zeros(2, 1, 16, 4, dtype=torch.bfloat16)
    for text, call in (
            ("uint8", lambda: ops.KV4Cache(k.float(), k, s)),
            ("head_dim", lambda: ops.KV4Cache(k[..., :16], k[..., :16], s)),
            ("scales", lambda: ops.KV4Cache(k, k, s[..., :2])),
            ("weights", lambda: ops.KV4Cache(k, k, s, torch.zeros(2, 1, 15))),
            ("contiguous", lambda: ops.KV4Cache(k[:, :, ::2], k[:, :, ::2], s[:, :, ::2])),
            ("at least one", lambda: ops.KV4Cache(k[:0], k[:0], s[:0])),
            ("CUDA device", lambda: ops.KV4Cache(k, k, s))):
        with pytest.raises(ValueError, match=text):
            call()


def test_no_read_only_loads(root):
    """The operators' kernels may begin while the kernel before them still writes their operands, and attend's
    output may be its query: the read-only path promises memory that does not change during a kernel."""
    folder = os.path.join(root, "compress-zip_b200", "csrc")
    names = [n for n in os.listdir(folder) if n.startswith("ops_")]
    assert len(names) >= 5
    for name in names:
        text = re.sub(r"//[^\n]*", "", open(os.path.join(folder, name)).read())
        assert not re.search(r"__ldg\w*\s*\(|\.global\.nc|\bconst\s+\w+\s*\*\s*__restrict__", text), name


def test_budgets_beyond_an_int(ops):
    """2^32 + 1 would reach the library as 1."""
    c = object.__new__(ops.KV4Cache)
    c._index, c.weights = -1, torch.zeros(1)
    n = torch.zeros(1, dtype=torch.int32)
    for budget, recent in ((1 << 31, 0), ((1 << 32) + 1, 0), (0, 0), (5, 6), (5, -1)):
        with pytest.raises(ValueError, match="budget"):
            c.evict(n, n, budget, recent)


def test_gradients_are_refused(ops):
    """There is no backward pass: a result without its gradient would be silent."""
    x, bias, scales = torch.zeros(4, 32), torch.zeros(8), torch.ones(8)
    codes = torch.zeros(8, 32, dtype=torch.int8)
    w = ops.QRows(codes, scales)

    def grad(t):
        return t.clone().requires_grad_()

    calls = [lambda: ops.linear_i8(grad(x), w), lambda: ops.linear_i8(grad(x).view(2, 2, 32), w), lambda: ops.linear_i8(x, w, bias=grad(bias)),
             lambda: ops.linear_i8(x, ops.QRows(codes, grad(scales))), lambda: ops.linear_i8(ops.QRows(codes, grad(scales)), w)]
    c = object.__new__(ops.KV4Cache)
    c._index, c.n_heads, c.head_dim, c.capacity = -1, 2, 64, 100
    n, q = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    calls.append(lambda: c.attend(grad(q), n, n))
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
    for call in calls[:5]:        # without gradients the next check answers
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):
            call()


def test_few_rows_on_many_channels_take_two_kernels(ops):
    """One kernel quantises a few short rows in every tile of channels: not where tiles come in many waves."""
    L = ops.lib()
    for m, n, k, two in ((1, 512, 384, False), (8, 512, 2048, False), (16, 4096, 2048, False), (1, 32768, 384, False),
                         (1, 128000, 384, True), (1, 16384, 2048, True), (8, 128000, 2048, True), (2, 4096, 11264, True),
                         (17, 100, 100, True), (0, 512, 384, False), (1, 0, 384, False)):
        need = L.czg_linear_i8_dynamic_workspace(m, n, k)
        assert need == (m * ((k + 15) // 16 * 16) + (4 * m + 15) // 16 * 16 if two else 0)
        assert need >= L.czg_linear_i8_workspace(m, k) or n == 0


def test_attend_limit_of_rows(ops):
    c = cache(ops)

    def attend(t):
        return ("czg_kv4_attend", c, P, 256, 256, 64, BF16, P, P, 2, t, 4, 100, 0.1, 1 << 40, 256, 256, 64, P, 1 << 50, None)

    refused(ops, E_LIMIT, "65,535 blocks", *attend(32768 * 8))      # 2 key heads of 32,768 blocks of 16 rows
    refused(ops, E_LIMIT, "too many rows", *attend(1 << 30))
    need = ops.lib().czg_kv4_attend_workspace        # with weights, scores; with several blocks of rows, partial results
    assert need(c, 2, 7, 4, 100) == 2 * 7 * 4 * 100 * 4
    assert need(c, 2, 9, 4, 100) == 2 * 2 * 32 * (64 * 4 + 16) + 2 * 9 * 4 * 100 * 4
    assert need(cache(ops, weights=None), 2, 9, 4, 100) == 0
