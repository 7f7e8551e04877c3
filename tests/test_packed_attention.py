"""Attention over packed documents (h3k_attention_packed) against a float64 softmax over exactly the keys that each row may
see: refusals on the CPU, the kernel on a B200, alone and in the chain of 4-bit calls that a block makes."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import h3b200 as H
from oracle import fp4_oracle as F4

BASE = 1 << 20  # an address that is aligned and never read
TYPES = {"bf16": (torch.bfloat16, H.BF16, 2.0 ** -8), "f16": (torch.float16, H.F16, 2.0 ** -11)}


def stream():
    return torch.cuda.current_stream().cuda_stream


def sync():
    H.check(H.lib().h3k_check(ctypes.c_void_p(stream())))


# ------------------------------------------------------------------------------------------------------- on the CPU

GOOD = dict(q=BASE, k=BASE, v=BASE, out=BASE, q_stride=512, k_stride=512, v_stride=512, out_stride=512, type=H.BF16, heads=4, kv_heads=4, head_dim=128,
            q_rows=9, k_rows=9, docs=2, prefix=3, q_start=BASE, k_start=BASE, scale=0.1)


@pytest.mark.parametrize("change,text", [
    (dict(type=H.F32), "bf16 or f16"), (dict(type=-1), "bf16 or f16"), (dict(head_dim=96), "64 or 128"), (dict(heads=0), "multiple"),
    (dict(kv_heads=0), "multiple"), (dict(heads=6), "multiple"), (dict(heads=65, kv_heads=1, q_stride=65 * 128, out_stride=65 * 128), "multiple"),
    (dict(q_rows=-1), "negative"), (dict(k_rows=-1, prefix=0), "negative"), (dict(docs=-1), "negative"), (dict(prefix=-1), "prefix"), (dict(prefix=10), "prefix"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(out=None), "null"), (dict(q_start=None), "null"), (dict(k_start=None), "null"),
    (dict(q=BASE + 8), "aligned"), (dict(out=BASE + 2), "aligned"), (dict(q_start=BASE + 2), "aligned"),
    (dict(q_stride=504), "overlap"), (dict(k_stride=516), "overlap"), (dict(v_stride=0), "overlap"), (dict(out_stride=511), "overlap")])
def test_refuses(change, text):
    a = H.h3k_packed_args(**(GOOD | change))
    assert H.lib().h3k_attention_packed(ctypes.byref(a), None) == H.H3_ERR_ARG
    assert text in H.lib().h3_last_error().decode()


def test_refuses_no_arguments_and_does_nothing_without_rows():
    assert H.lib().h3k_attention_packed(None, None) == H.H3_ERR_ARG
    for change in (dict(q_rows=0), dict(docs=0)):
        a = H.h3k_packed_args(**(GOOD | change))
        assert H.lib().h3k_attention_packed(ctypes.byref(a), None) == H.H3_OK


def test_the_binding_has_the_headers_struct(tmp_path):
    names = [f[0] for f in H.h3k_packed_args._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "h3_c.h"\nint main(void) { printf("%zu", sizeof(h3k_packed_args));\n'
                   + "".join(f'printf(" %zu", offsetof(h3k_packed_args, {n}));\n' for n in names) + "return 0; }\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(H.h3k_packed_args)] + [getattr(H.h3k_packed_args, n).offset for n in names]


# ---------------------------------------------------------------------------------------------------------- on a B200

def starts(lengths, first=0):
    s = [first]
    for n in lengths:
        s.append(s[-1] + n)
    return s


def call(q, k, v, out, q_start, k_start, prefix, scale=0.0, check=True):
    """q [rows][heads][dim], k and v [rows][kv][dim] (views may have wider rows), starts on the GPU."""
    t = {v_[0]: v_[1] for v_ in TYPES.values()}[q.dtype]
    a = H.h3k_packed_args(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0),
                          out_stride=out.stride(0), type=t, heads=q.shape[1], kv_heads=k.shape[1], head_dim=q.shape[2], q_rows=q.shape[0], k_rows=k.shape[0],
                          docs=q_start.numel() - 1, prefix=prefix, q_start=q_start.data_ptr(), k_start=k_start.data_ptr(), scale=scale)
    H.check(H.lib().h3k_attention_packed(ctypes.byref(a), stream()))
    if check:
        sync()


def expected(q, k, v, q_start, k_start, prefix, scale, before):
    """(want, how far the kernel may be off), float64. Off: every probability is rounded to the type (eps) and off by its
    score's error relatively (an fp32 sum of dim products and three fp32 operations on the score), numerator and sum alike;
    fp16 probabilities below 2^-14 are off by up to 2^-25 (the largest is at least 1); the result is rounded once."""
    eps = TYPES[[n for n, t in TYPES.items() if t[0] == q.dtype][0]][2]
    want, tol = before.double().clone(), torch.zeros(before.shape, dtype=torch.float64, device=before.device)
    dim, group = q.shape[2], q.shape[1] // k.shape[1]
    for d in range(len(q_start) - 1):
        rows = slice(q_start[d], q_start[d + 1])
        keys = torch.tensor(sorted(set(range(prefix)) | set(range(k_start[d], k_start[d + 1]))), dtype=torch.int64, device=q.device)
        if rows.start == rows.stop:
            continue
        if not len(keys):
            want[rows] = 0
            continue
        for h in range(q.shape[1]):
            Q, K, V = q[rows, h].double(), k[keys, h // group].double(), v[keys, h // group].double()
            s = Q @ K.T * scale
            w = torch.softmax(s, 1)
            reach = (Q.norm(dim=1)[:, None] * K.norm(dim=1)[None]).amax(1, keepdim=True) * scale
            relative = 2 * (dim + 8) * 2.0 ** -23 * reach + 2.0 ** -18
            o = w @ V
            want[rows, h] = o
            tol[rows, h] = (w @ V.abs()) * (eps + relative) + eps * o.abs()
            if q.dtype == torch.float16:
                tol[rows, h] += len(keys) * 2.0 ** -25 * V.abs().max() + 2.0 ** -25
    return want, tol


def compare(out, want, tol):
    off = (out.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (bad.nonzero()[:5], off[bad][:5], tol[bad][:5])


SELF = [([1], 0), ([1, 1, 1], 0), ([1, 1, 1], 1), ([5, 0, 130, 0], 5), ([256, 257, 3], 0), ([77, 300, 128, 64, 1000], 77), ([200, 1, 55, 129, 127], 200), ([0, 0, 7], 0),
        ([128, 128, 384], 128), ([3] * 70, 3), ([1] * 1100, 0),
        ([40] + [200] * 33 + [700, 0, 1], 40), ([5, 3000, 17, 1111, 640], 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,prefix", SELF, ids=[f"{len(s[0])}docs{sum(s[0])}rows{s[1]}prefix" for s in SELF])
def test_self_attention_of_documents(cuda, type, dim, lengths, prefix):
    """q, k and v as one [rows][3][heads][dim] tensor; the prefix's rows are the first document; spare rows behind hold NaN."""
    heads, total, spare = 3, sum(lengths), 21
    g = torch.Generator(device=cuda).manual_seed(total)
    qkv = torch.randn(total + spare, 3, heads, dim, generator=g, device=cuda).to(TYPES[type][0])
    qkv[total:] = float("nan")
    q, k, v = qkv.unbind(1)
    out = torch.full((total + spare, heads, dim), 7.0, device=cuda, dtype=qkv.dtype)
    before, s = out.clone(), starts(lengths)
    at = torch.tensor(s, dtype=torch.int32, device=cuda)
    call(q, k, v, out, at, at, prefix)
    compare(out, *expected(q, k, v, s, s, prefix, dim ** -0.5, before))


CROSS = [([1], [1], 0), ([1], [9000], 0), ([1], [33024], 0), ([300], [2500], 0), ([2, 0, 1, 3], [0, 300, 7, 129], 0), ([2, 5, 1, 3], [0, 300, 0, 129], 130), ([40, 1, 260], [4000, 0, 5000], 1000),
         ([1] * 9, [1024] * 9, 0), ([4], [0], 0), ([4], [0], 700)]


@pytest.mark.gpu
@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("heads,kv", [(2, 2), (6, 2), (7, 1), (10, 2), (33, 1), (64, 1)])
@pytest.mark.parametrize("q_len,k_len,prefix", CROSS, ids=[f"{sum(c[0])}on{sum(c[1])}prefix{c[2]}" for c in CROSS])
def test_shared_kv_heads_and_long_keys(cuda, type, heads, kv, q_len, k_len, prefix):
    """Few query rows on long keys (split over a cluster), documents without keys, wider rows, rows before the first document."""
    dim = 128 if heads % 2 == 0 else 64
    lead, spare = 3, 5
    q_start, k_start = starts(q_len, lead), starts(k_len, prefix + (lead if prefix else 0))
    nq, nk = q_start[-1] + spare, max(k_start[-1], prefix) + spare
    g = torch.Generator(device=cuda).manual_seed(nq + nk)
    t = TYPES[type][0]
    q = torch.randn(nq, heads + 1, dim, generator=g, device=cuda).to(t)[:, :heads]
    k, v = (torch.randn(nk, kv + i, dim, generator=g, device=cuda).to(t)[:, :kv] for i in (0, 2))
    seen = torch.zeros(nk, dtype=torch.bool, device=cuda)
    seen[:prefix] = True
    seen[k_start[0]:k_start[-1]] = True
    k[~seen], v[~seen] = float("nan"), float("inf")
    out = torch.full((nq, heads + 2, dim), 7.0, device=cuda, dtype=t)
    before = out.clone()
    at_q, at_k = (torch.tensor(s, dtype=torch.int32, device=cuda) for s in (q_start, k_start))
    call(q, k, v, out[:, :heads], at_q, at_k, prefix, scale=0.2)
    compare(out[:, :heads], *expected(q, k, v, q_start, k_start, prefix, 0.2, before[:, :heads]))
    assert torch.equal(out[:, heads:], before[:, heads:])


@pytest.mark.gpu
@pytest.mark.parametrize("split", [False, True])
def test_what_other_documents_hold_does_not_reach_a_row(cuda, split):
    """NaN and infinities in one document's keys and values: its own rows show them, no other row changes by a bit."""
    lengths = [600, 1000, 700] if split else [130, 200, 90] * 9
    heads, dim = 2 if split else 20, 128
    s = starts(lengths)
    at = torch.tensor(s, dtype=torch.int32, device=cuda)
    qkv = torch.randn(s[-1], 3, heads, dim, device=cuda).bfloat16()
    clean, dirty = (torch.zeros(s[-1], heads, dim, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    call(*qkv.unbind(1), clean, at, at, 0)
    qkv[s[1]:s[2]:3, 1] = float("nan")
    qkv[s[1]:s[2]:2, 2] = float("inf")
    call(*qkv.unbind(1), dirty, at, at, 0)
    rows = torch.ones(s[-1], dtype=torch.bool, device=cuda)
    rows[s[1]:s[2]] = False
    assert torch.equal(dirty[rows], clean[rows])
    assert torch.isnan(dirty[~rows]).all()


@pytest.mark.gpu
def test_scores_far_apart_and_at_minus_infinity(cuda):
    """Scores of +-1000s (one key takes all), a running maximum that grows block by block, and rows whose every score is -infinity."""
    rows, keys, dim = 40, 700, 64
    g = torch.Generator(device=cuda).manual_seed(1)
    q = torch.randn(rows, 1, dim, generator=g, device=cuda).bfloat16() * 30
    k = torch.randn(keys, 1, dim, generator=g, device=cuda).bfloat16() * torch.linspace(0.1, 30, keys, device=cuda)[:, None, None].bfloat16()
    v = torch.randn(keys, 1, dim, generator=g, device=cuda).bfloat16()
    out = torch.zeros_like(q)
    at_q, at_k = (torch.tensor([0, n], dtype=torch.int32, device=cuda) for n in (rows, keys))
    call(q, k, v, out, at_q, at_k, 0)
    # Here the score's own error (reach x 2^-23 x dim) is what counts: the bound allows it.
    compare(out, *expected(q, k, v, [0, rows], [0, keys], 0, dim ** -0.5, out))
    q = torch.ones(rows, 1, dim, device=cuda).bfloat16()
    k[:] = float("-inf")
    call(q, k, v, out, at_q, at_k, 0)
    assert (out == 0).all()


@pytest.mark.gpu
def test_rows_far_apart_in_memory(cuda):
    """Offsets past 32 bits: rows 2^27 elements apart."""
    rows, dim, stride = 40, 64, 1 << 27
    big = torch.empty(stride * (rows - 1) + 3 * dim, dtype=torch.bfloat16, device=cuda)
    q, k, v = (big.as_strided((rows, 1, dim), (stride, dim, 1), i * dim) for i in range(3))
    for t in (q, k, v):
        t.copy_(torch.randn(rows, 1, dim, device=cuda))
    at = torch.tensor([0, 17, 40], dtype=torch.int32, device=cuda)
    want, tol = expected(q.contiguous(), k.contiguous(), v.contiguous(), [0, 17, 40], [0, 17, 40], 2, dim ** -0.5, q.contiguous())
    out = torch.zeros(rows, 1, dim, device=cuda, dtype=torch.bfloat16)
    call(q, k, v, out, at, at, 2)
    compare(out, want, tol)
    far = big.as_strided((rows, 1, dim), (stride, dim, 1), 0)
    call(out.clone(), out.clone(), out.clone(), far, at, at, 2)
    near = torch.zeros_like(out)
    call(out.clone(), out.clone(), out.clone(), near, at, at, 2)
    assert torch.equal(far.contiguous(), near)


@pytest.mark.gpu
@pytest.mark.parametrize("q_start,k_start", [([0, 10, 5, 20], [0, 10, 15, 20]), ([0, 10, 15, 21], [0, 10, 15, 20]), ([-3, 10, 15, 20], [0, 10, 15, 20]),
                                             ([0, 10, 15, 20], [0, 10, 15, 30]), ([0, 10, 15, 20], [0, -7, 15, 20]), ([0, 10, 15, 2 ** 31 - 1], [0, 2 ** 31 - 1, 15, 20])])
def test_bad_starts_are_a_device_error(cuda, q_start, k_start):
    q, k, v = (torch.randn(20, 2, 64, device=cuda).half() for _ in range(3))
    whole = torch.full((24, 2, 64), 7.0, device=cuda).half()
    at_q, at_k = (torch.tensor(s, dtype=torch.int32, device=cuda) for s in (q_start, k_start))
    call(q, k, v, whole[2:22], at_q, at_k, 4, check=False)
    assert H.lib().h3k_check(ctypes.c_void_p(stream())) == H.H3_ERR_DEVICE
    assert (whole[:2] == 7).all() and (whole[22:] == 7).all()
    sync()  # the error is reported once


@pytest.mark.gpu
def test_a_replayed_graph_sees_new_starts_and_two_streams_agree(cuda):
    heads, dim, rows = 4, 128, 900
    q, k, v = (torch.randn(rows, heads, dim, device=cuda).bfloat16() for _ in range(3))
    out = torch.zeros_like(q)
    first, second = [0, 100, 512, 900, 900], [0, 300, 301, 640, 900]
    at = torch.tensor(first, dtype=torch.int32, device=cuda)
    call(q, k, v, out, at, at, 100)
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(q, k, v, out, at, at, 100, check=False)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    at.copy_(torch.tensor(second, dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    compare(out, *expected(q, k, v, second, second, 100, dim ** -0.5, out))
    want, outs = out.clone(), []
    torch.cuda.synchronize()
    for _ in range(2):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            outs.append(torch.zeros_like(q))
            call(q, k, v, outs[-1], at, at, 100, check=False)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    sync()


@pytest.mark.gpu
@pytest.mark.parametrize("f", [F4.MX, F4.NV])
def test_the_attention_half_of_a_block_on_packed_documents_in_4_bits(cuda, f):
    """x -> quantise -> q/k/v product -> attention per document -> quantise -> out product and gated residual, queued without a
    wait; then every stage is checked against float64 on what the stage before it left."""
    lengths, prefix, heads, dim = [40, 333, 1, 150], 40, 4, 512
    rows, inner, s = sum(lengths), 4 * 128, starts(lengths)
    g = torch.Generator(device=cuda).manual_seed(f)
    L = H.lib()
    h = torch.randn(rows, dim, generator=g, device=cuda).bfloat16()
    w_qkv, w_out = (torch.randn(n, k, generator=g, device=cuda).bfloat16() * 0.05 for n, k in ((3 * inner, dim), (dim, inner)))
    wq, wk = (1 + 0.1 * torch.randn(128, generator=g, device=cuda) for _ in range(2))
    angle = torch.rand(rows, 48, generator=g, device=cuda) * 6.28
    rope = torch.stack([angle.cos(), angle.sin()], 2).contiguous()
    mod = torch.randn(2, 6, dim, generator=g, device=cuda)
    idx = (torch.arange(rows, device=cuda) % 2).to(torch.uint8)
    x = torch.randn(rows, dim, generator=g, device=cuda)
    before = x.clone()
    at = torch.tensor(s, dtype=torch.int32, device=cuda)

    def quantise(t):
        codes, tiles = (torch.empty(n, dtype=torch.uint8, device=cuda) for n in H.fp4_sizes(*t.shape, f))
        row = torch.empty(t.shape[0], device=cuda) if f == F4.NV else None
        H.check(L.h3k_quant_rows_fp4(t.data_ptr(), H.BF16, t.stride(0), *t.shape, f, codes.data_ptr(), tiles.data_ptr(), None if row is None else row.data_ptr(), stream()))
        return codes, tiles, row

    def product(A, B, m, n, k, epi, **kw):
        a = H.h3k_gemm_args(M=m, N=n, K=k, a_scale=None if A[2] is None else A[2].data_ptr(), b_scale=None if B[2] is None else B[2].data_ptr(), eps=1e-6, **kw)
        H.check(L.h3k_gemm_fp4(A[0].data_ptr(), A[1].data_ptr(), B[0].data_ptr(), B[1].data_ptr(), f, ctypes.byref(a), epi, stream()))

    qkv = torch.zeros(rows, 3, heads, 128, dtype=torch.bfloat16, device=cuda)
    o = torch.zeros(rows, heads, 128, dtype=torch.bfloat16, device=cuda)
    B1, B2, A1 = quantise(w_qkv), quantise(w_out), quantise(h)
    product(A1, B1, rows, 3 * inner, dim, H.EPI_QKV, out=qkv.data_ptr(), rope=rope.data_ptr(), qn_w=wq.data_ptr(), kn_w=wk.data_ptr(), inner=inner, heads_per_rank=heads,
            rows_local=rows)
    call(*qkv.unbind(1), o, at, at, prefix, check=False)
    A2 = quantise(o.view(rows, inner))
    product(A2, B2, rows, dim, inner, H.EPI_GATE_RESID, x=x.data_ptr(), ldx=dim, mod=mod.data_ptr(), mod_idx=idx.data_ptr(), gate_slot=2, dim=dim)
    sync()

    def values(t, n):
        codes, bytes_ = F4.unpack(t[0].view(n, -1).cpu().numpy(), t[1].cpu().numpy(), f)
        return torch.from_numpy(F4.values(codes, bytes_, None if t[2] is None else t[2].cpu().numpy(), f)).to(cuda)

    # v of the q/k/v product (q and k have a test of their own), bf16
    want = (values(A1, rows) @ values(B1, 3 * inner)[2 * inner:].T).view(rows, heads, 128)
    sums = (values(A1, rows).abs() @ values(B1, 3 * inner)[2 * inner:].abs().T).view(rows, heads, 128)
    assert ((qkv[:, 2] - want).abs() <= 2.0 ** -8 * want.abs() + (dim + 4) * 2.0 ** -23 * sums).all()
    compare(o, *expected(*qkv.unbind(1), s, s, prefix, 128 ** -0.5, o))
    y = values(A2, rows) @ values(B2, dim).T
    gate = mod[idx.long(), 2].double()
    sums = values(A2, rows).abs() @ values(B2, dim).abs().T
    want = before.double() + gate * y
    assert ((x - want).abs() <= gate.abs() * (inner + 4) * 2.0 ** -23 * sums + 2.0 ** -23 * (want.abs() + (gate * y).abs())).all()


# documents x (query rows, keys): few and many rows on few and many keys, where one kernel or another, and whole or split runs, are the fastest
MIXES = [(24, 64, 60), (24, 4, 300), (3, 200, 40), (4, 8, 4000), (3, 64, 6000), (16, 16, 2000), (1, 64, 6000), (60, 20, 300), (3, 600, 1500), (9, 130, 900)]


@pytest.mark.gpu
@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("heads,kv,dim", [(6, 6, 64), (3, 3, 128), (8, 2, 128), (16, 1, 64), (20, 1, 128)])
@pytest.mark.parametrize("docs,rows,keys", MIXES)
def test_every_kind_of_batch(cuda, type, heads, kv, dim, docs, rows, keys):
    """Uneven documents around those averages, one of them without keys of its own."""
    rng = np.random.default_rng(docs + rows + keys)
    q_start, k_start = (starts(np.maximum(1, rng.uniform(0.3, 1.7, docs) * n).astype(int).tolist(), lead) for n, lead in ((rows, 0), (keys, 70)))
    if docs > 2:
        k_start[2] = k_start[1]
    g = torch.Generator(device=cuda).manual_seed(rows)
    q, k, v = (torch.randn(n, h, dim, generator=g, device=cuda).to(TYPES[type][0]) for n, h in ((q_start[-1], heads), (k_start[-1], kv), (k_start[-1], kv)))
    out = torch.full_like(q, 7.0)
    before = out.clone()
    at_q, at_k = (torch.tensor(s, dtype=torch.int32, device=cuda) for s in (q_start, k_start))
    call(q, k, v, out, at_q, at_k, 70)
    compare(out, *expected(q, k, v, q_start, k_start, 70, dim ** -0.5, before))


FIRST = """
import ctypes, sys, torch
import h3b200 as H
sys.path.insert(0, {tests!r})
import test_packed_attention as T
dev = torch.device("cuda")
q, k, v = (torch.randn(n, 2, 128, device=dev).bfloat16() for n in ({rows}, {keys}, {keys}))
out, again = torch.zeros_like(q), torch.zeros_like(q)
at_q, at_k = (torch.tensor([0, n], dtype=torch.int32, device=dev) for n in ({rows}, {keys}))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    T.call(q, k, v, out, at_q, at_k, 0, check=False)
graph.replay()
torch.cuda.synchronize()
T.call(q, k, v, again, at_q, at_k, 0)
assert torch.equal(out, again) and out.abs().sum() > 0
"""


@pytest.mark.gpu
@pytest.mark.parametrize("rows,keys", [(1, 9000), (40, 50), (900, 900)])
def test_the_first_call_of_a_process_may_be_captured(cuda, rows, keys):
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.join(here, "..", "mako-video_b200"), os.path.join(here, ".."), os.environ.get("PYTHONPATH", "")]))
    r = subprocess.run([sys.executable, "-c", FIRST.format(tests=here, rows=rows, keys=keys)], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


# ------------------------------------------------------------------------- who hears of starts that are not in order

def test_refuses_a_status_word_that_is_not_aligned():
    a = H.h3k_packed_args(**(GOOD | dict(status=BASE + 2)))
    assert H.lib().h3k_attention_packed(ctypes.byref(a), None) == H.H3_ERR_ARG
    assert "aligned" in H.lib().h3_last_error().decode()


def queue(q_start, k_start, status=None, rows=20):
    """A call on `rows` rows of 2 heads of 64, not waited for; what it uses is returned, to be kept."""
    q, k, v = (torch.randn(rows, 2, 64, device="cuda").half() for _ in range(3))
    out = torch.zeros_like(q)
    at = [torch.tensor(s, dtype=torch.int32, device="cuda") if isinstance(s, list) else s for s in (q_start, k_start)]
    a = H.h3k_packed_args(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), q_stride=128, k_stride=128, v_stride=128, out_stride=128, type=H.F16,
                          heads=2, kv_heads=2, head_dim=64, q_rows=rows, k_rows=rows, docs=at[0].numel() - 1, q_start=at[0].data_ptr(), k_start=at[1].data_ptr(),
                          **({} if status is None else dict(status=status.data_ptr())))
    H.check(H.lib().h3k_attention_packed(ctypes.byref(a), stream()))
    return q, k, v, out, at


BAD, FINE = [0, 10, 5, 20], [0, 10, 15, 20]


@pytest.mark.gpu
def test_a_step_beside_a_call_with_bad_starts_is_not_told_of_them(cuda):
    """The steps and decodes of others on the device end well, and the caller still hears of the starts."""
    from test_step_gpu import MINI, MINI_LAYOUT, inputs
    lay, text, video, audio = inputs(MINI_LAYOUT, MINI)
    m = H.Model(MINI, seed=1)
    m.begin(text, lay)
    want = m.step(video, audio, 0.7, 0.4)
    keep = queue(BAD, FINE)
    torch.cuda.synchronize()
    got = m.step(video, audio, 0.7, 0.4)
    m.synchronize()
    m.close()
    assert all(np.array_equal(g, w) for g, w in zip(got, want))
    assert H.lib().h3k_wait_selftest(1_000_000, stream()) == H.H3_ERR_DEVICE  # a failure of its own, reported and cleared
    assert H.lib().h3k_check(ctypes.c_void_p(stream())) == H.H3_ERR_DEVICE
    assert "starts" in H.lib().h3_last_error().decode()
    sync()
    del keep


@pytest.mark.gpu
def test_each_caller_has_a_status_word_of_its_own(cuda):
    """Two callers on two streams, one with bad starts: its word says so, the other's and h3k_check do not. A word is written by every run."""
    words = torch.full((4,), -1, dtype=torch.int32, device=cuda)
    keep = []
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    for side, word, q_start in ((sides[0], words[0:1], BAD), (sides[1], words[1:2], FINE)):
        with torch.cuda.stream(side):
            keep.append(queue(q_start, FINE, word))
    torch.cuda.synchronize()
    assert words.tolist() == [1, 0, -1, -1]
    sync()
    keep.append(queue(FINE, [0, 10, 15, 21], words[0:1]))
    keep.append(queue([0] * 40 + [20], [0] * 41, words[2:3]))
    keep.append(queue([0], [0], words[3:4]))  # no document: nothing to find
    torch.cuda.synchronize()
    assert words.tolist() == [1, 0, 0, 0]
    sync()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [20, 700])
def test_a_status_word_follows_the_starts_of_a_replayed_graph(cuda, rows):
    word = torch.zeros(1, dtype=torch.int32, device=cuda)
    at = torch.tensor([0, 3, 9, rows], dtype=torch.int32, device=cuda)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep = queue(at, at, word, rows)
    for starts_now, want in (([0, 3, 9, rows], 0), ([0, 9, 3, rows], 1), ([0, 3, 9, rows + 1], 1), ([0, 0, 0, 0], 0)):
        at.copy_(torch.tensor(starts_now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert word.item() == want
    sync()
    del keep


@pytest.mark.parametrize("docs", [2 ** 30 + 1, 2 ** 31 - 33, 2 ** 31 - 1])
def test_refuses_more_documents_than_the_lookup_can_number(docs):
    a = H.h3k_packed_args(**(GOOD | dict(q_rows=1, kv_heads=4, docs=docs)))
    assert H.lib().h3k_attention_packed(ctypes.byref(a), None) == H.H3_ERR_ARG
    assert "documents" in H.lib().h3_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("docs,rows,keys", [(1, 1, 40), (1, 1, 9000), (40, 30, 60), (3, 300, 200), (3, 40, 5000), (2, 600, 2000)])
def test_rows_whose_scores_are_all_minus_infinity_are_zeros_whatever_the_values(cuda, type, dim, docs, rows, keys):
    """The even documents' keys are -infinity and their values infinities and NaNs; the odd ones' rows are as ever."""
    q_start, k_start = starts([rows] * docs), starts([keys] * docs)
    g = torch.Generator(device=cuda).manual_seed(rows)
    q, k, v = (torch.randn(n, 2, dim, generator=g, device=cuda).to(TYPES[type][0]) for n in (docs * rows, docs * keys, docs * keys))
    q, out = q.abs() + 0.1, torch.full_like(q, 7.0)
    for d in range(0, docs, 2):
        k[k_start[d]:k_start[d + 1]] = float("-inf")
        v[k_start[d]:k_start[d + 1]:2], v[k_start[d] + 1:k_start[d + 1]:2] = float("inf"), float("nan")
    at_q, at_k = (torch.tensor(s, dtype=torch.int32, device=cuda) for s in (q_start, k_start))
    call(q, k, v, out, at_q, at_k, 0)
    out, q, k, v = (t.view(docs, -1, 2, dim) for t in (out, q, k, v))
    assert (out[0::2] == 0).all()
    for d in range(1, min(docs, 4), 2):
        compare(out[d], *expected(q[d], k[d], v[d], [0, rows], [0, keys], 0, dim ** -0.5, out[d]))
