"""Microscaled 4-bit rows (h3k_quant_rows_fp4, h3k_dequant_rows_fp4, h3k_gemm_fp4) against float64 restatements: the
refusals and the oracle's own checks on the CPU, the kernels on a B200."""
import ctypes

import numpy as np
import pytest
import torch

import h3b200 as H
from oracle import fp4_oracle as F4

FORMATS = [F4.MX, F4.NV]
TYPES = {"bf16": (torch.bfloat16, H.BF16), "f16": (torch.float16, H.F16), "f32": (torch.float32, H.F32)}
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def p(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def sync():
    H.check(H.lib().h3k_check(ctypes.c_void_p(stream())))


# ------------------------------------------------------------------------------------------------------- on the CPU

def test_nearest_value_ties_go_to_the_even_code():
    ties = [(0.25, 0), (0.75, 2), (1.25, 2), (1.75, 4), (2.5, 4), (3.5, 6), (5.0, 6), (7.9, 7), (0.2500001, 1), (0.7499999, 1)]
    got = F4.nearest(np.array([t[0] for t in ties]), F4.VALUES)
    assert got.tolist() == [t[1] for t in ties]


@pytest.mark.parametrize("f", FORMATS)
def test_oracle_packing_is_its_own_inverse_and_the_layout_is_as_documented(f):
    x = np.random.default_rng(f).standard_normal((200, 160))
    codes, bytes_, row, _ = F4.quantise(x, f)
    packed, tiles = F4.pack(codes, bytes_)
    c2, b2 = F4.unpack(packed, tiles, f)
    np.testing.assert_array_equal(c2, codes)
    np.testing.assert_array_equal(b2, bytes_)
    r, j = 133, bytes_.shape[1] - 1
    kt = -(-bytes_.shape[1] // 4)
    assert tiles[((r // 128) * kt + j // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + j % 4] == bytes_[r, j]
    # the largest of a block is in [4, 8) (mx) or within an e4m3 step of 6 (nv) of its scales, so a value is off by 2 of them
    # (mx: 8 becomes 6) or 1.2 (half the widest step, and 6 / (1 - 1/16) becomes 6), and they are at most a fourth of it
    most = np.repeat(np.abs(x.reshape(200, -1, F4.BLOCK[f])).max(2), F4.BLOCK[f], 1)
    assert (np.abs(F4.values(codes, bytes_, row, f) - x) <= (2.0 if f == F4.MX else 1.2) * most / 4).all()


@pytest.mark.parametrize("rows,K,f,want", [(1, 32, F4.MX, (16, 512)), (1, 32, F4.NV, (16, 512)), (128, 128, F4.MX, (8192, 512)), (129, 160, F4.MX, (10320, 2048)),
                                           (129, 160, F4.NV, (10320, 3 * 1024)), (0, 64, F4.NV, (0, 0)), (33024, 5120, F4.NV, (33024 * 2560, 258 * 80 * 512))])
def test_sizes(rows, K, f, want):
    assert H.fp4_sizes(rows, K, f) == want


BASE = 1 << 20  # an address that is aligned and never read: every call below is refused before any device work


def refused(rc, text):
    assert rc == H.H3_ERR_ARG
    assert text in H.lib().h3_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(format=2), "unknown format"), (dict(type=3), "unknown element type"), (dict(K=48), "multiple of 32"), (dict(K=0), "multiple of 32"),
    (dict(rows=-1), "negative"), (dict(x=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(row_scale=None), "row_scale"),
    (dict(format=0), "row_scale"), (dict(ldx=68), "16 bytes"), (dict(x=BASE + 2), "not aligned"), (dict(codes=BASE + 8), "not aligned")])
def test_quantise_refuses(change, text):
    a = dict(x=BASE, type=H.BF16, ldx=64, rows=3, K=64, format=F4.NV, codes=BASE, scales=BASE, row_scale=BASE) | change
    refused(H.lib().h3k_quant_rows_fp4(a["x"], a["type"], a["ldx"], a["rows"], a["K"], a["format"], a["codes"], a["scales"], a["row_scale"], None), text)


@pytest.mark.parametrize("change,text", [
    (dict(format=-1), "unknown format"), (dict(type=-1), "unknown element type"), (dict(K=16), "multiple of 32"), (dict(out=None), "null"),
    (dict(ldo=56), "overlap"), (dict(ldo=68), "16 bytes"), (dict(out=BASE + 4), "not aligned")])
def test_dequantise_refuses(change, text):
    a = dict(codes=BASE, scales=BASE, rows=3, K=64, format=F4.MX, type=H.BF16, out=BASE, ldo=64) | change
    refused(H.lib().h3k_dequant_rows_fp4(a["codes"], a["scales"], None, a["rows"], a["K"], a["format"], a["type"], a["out"], a["ldo"], None), text)


@pytest.mark.parametrize("epi,change,text", [
    (H.EPI_BF16, dict(N=20), "multiple of 8"), (H.EPI_BF16, dict(K=72), "multiple of 32"), (H.EPI_BF16, dict(M=-2), "negative"),
    (H.EPI_BF16, dict(lda=128), "contiguous"), (H.EPI_BF16, dict(a_chunks=2), "contiguous"), (H.EPI_BF16, dict(out=None), "output"),
    (H.EPI_BF16, dict(ldo=248), "overlap"), (H.EPI_BF16, dict(ldo=260), "16 bytes"), (H.EPI_F32, dict(ldo=258), "16 bytes"),
    (H.EPI_S32, {}, "epilogue"), (9, {}, "epilogue"), (H.EPI_SWIGLU, dict(N=264), "256-row"), (H.EPI_SWIGLU, dict(ldo=120), "overlap"),
    (H.EPI_QKV, dict(N=768, inner=256, heads_per_rank=2, rows_local=1, rope=BASE, qn_w=BASE, kn_w=BASE), "rows"),
    (H.EPI_QKV, dict(N=768, inner=128, heads_per_rank=1, rows_local=3), "inner"),
    (H.EPI_QKV, dict(N=768, inner=256, heads_per_rank=2, rows_local=3), "rotary"),
    (H.EPI_GATE_RESID, {}, "mod_idx"), (H.EPI_GATE_RESID, dict(x=BASE, ldx=256, mod=BASE, mod_idx=BASE, gate_slot=6, dim=256), "slot"),
    (H.EPI_GATE_RESID, dict(x=BASE, ldx=256, mod=BASE, mod_idx=BASE, gate_slot=2, dim=128), "width"),
    (H.EPI_BF16, dict(bias=BASE + 4), "not aligned"), (H.EPI_BF16, dict(b_scale=BASE + 4), "not aligned")])
def test_product_refuses(epi, change, text):
    a = H.h3k_gemm_args(**(dict(M=3, N=256, K=64, out=BASE, ldo=256) | change))
    refused(H.lib().h3k_gemm_fp4(BASE, BASE, BASE, BASE, F4.MX, ctypes.byref(a), epi, None), text)


def test_product_refuses_null_operands_and_a_wrong_format():
    a = H.h3k_gemm_args(M=3, N=256, K=64, out=BASE, ldo=256)
    L = H.lib()
    refused(L.h3k_gemm_fp4(None, BASE, BASE, BASE, F4.MX, ctypes.byref(a), H.EPI_BF16, None), "null")
    refused(L.h3k_gemm_fp4(BASE, BASE, BASE, None, F4.MX, ctypes.byref(a), H.EPI_BF16, None), "null")
    refused(L.h3k_gemm_fp4(BASE, BASE, BASE, BASE, 7, ctypes.byref(a), H.EPI_BF16, None), "format")
    refused(L.h3k_gemm_fp4(BASE, BASE, BASE, BASE, F4.MX, None, H.EPI_BF16, None), "null")


def test_more_rows_than_whole_scale_tiles_can_number_are_refused():
    L, most = H.lib(), 0x7fffff80
    assert H.fp4_sizes(most, 32, F4.MX) == (most * 16, most // 128 * 512)
    refused(L.h3k_fp4_sizes(most + 1, 32, F4.MX, None, None), "rows")
    refused(L.h3k_quant_rows_fp4(BASE, H.BF16, 0, most + 1, 32, F4.MX, BASE, BASE, None, None), "rows")
    refused(L.h3k_dequant_rows_fp4(BASE, BASE, None, most + 1, 32, F4.MX, H.BF16, BASE, 32, None), "rows")
    for change, text in ((dict(M=most + 1), "rows"), (dict(N=most + 8), "columns")):
        a = H.h3k_gemm_args(**(dict(M=3, N=256, K=64, out=BASE, ldo=256) | change))
        refused(L.h3k_gemm_fp4(BASE, BASE, BASE, BASE, F4.MX, ctypes.byref(a), H.EPI_BF16, None), text)


def test_no_rows_is_no_work():
    L = H.lib()
    assert L.h3k_quant_rows_fp4(None, H.BF16, 64, 0, 64, F4.MX, None, None, None, None) == H.H3_OK
    assert L.h3k_dequant_rows_fp4(None, None, None, 0, 64, F4.MX, H.F32, None, 64, None) == H.H3_OK
    a = H.h3k_gemm_args(M=0, N=256, K=64, ldo=256)
    assert L.h3k_gemm_fp4(None, None, None, None, F4.MX, ctypes.byref(a), H.EPI_BF16, None) == H.H3_OK


# ---------------------------------------------------------------------------------------------------------- on a B200

def gpu_quantise(x, f, K=None, spare=0):
    """(codes, tiles, row scales) of x [rows][ld] on the GPU, the first K columns."""
    rows, K = x.shape[0], K or x.shape[1]
    cb, sb = H.fp4_sizes(rows, K, f)
    codes = torch.full((cb + spare,), 0xEE, dtype=torch.uint8, device=x.device)
    tiles = torch.full((sb + spare,), 0xEE, dtype=torch.uint8, device=x.device)
    row = torch.full((rows + spare,), -1.0, device=x.device) if f == F4.NV else None
    t = {v[0]: v[1] for v in TYPES.values()}[x.dtype]
    H.check(H.lib().h3k_quant_rows_fp4(p(x), t, x.stride(0), rows, K, f, p(codes), p(tiles), p(row), stream()))
    sync()
    return codes, tiles, row


def rows_like(rows, K, seed, kind="normal"):
    g = np.random.default_rng(seed)
    x = g.standard_normal((rows, K)) * np.exp(g.standard_normal((1, K)))
    if kind == "ties":  # multiples of the borders between codes, times powers of two
        x = g.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.25, -1.25, -5.0, 0.0], (rows, K)) * 2.0 ** g.integers(-3, 4, (rows, 1))
    if kind == "wide":  # magnitudes over the whole range, whole blocks and rows of zeros and of the smallest
        x *= 2.0 ** g.integers(-140, 120, (rows, 1))
        x[:, : K // 2] *= 2.0 ** -12.0
        x[0] = 0
        x[-1, :32] = 0
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("kind", ["normal", "ties", "wide"])
@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("rows,K,ld", [(1, 32, 32), (3, 96, 104), (130, 160, 160), (33, 2048, 2048), (5, 4160, 4224), (7, 8224, 8224), (2, 16416, 16416), (3, 40000, 40000)])
def test_quantise_bit_exact(cuda, f, kind, type, rows, K, ld):
    check_quantise(cuda, f, kind, type, rows, K, ld)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "wide"])
@pytest.mark.parametrize("type", ["bf16", "f16"])
@pytest.mark.parametrize("rows,K,ld", [(1201, 8224, 8232), (1201, 16384, 16384)])
def test_quantise_many_long_rows_bit_exact(cuda, kind, type, rows, K, ld):
    """Rows that CTAs walk instead of having one each."""
    check_quantise(cuda, F4.NV, kind, type, rows, K, ld)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,type,rows,K,ld", [("normal", "bf16", 1801, 16384, 16384), ("wide", "f16", 19001, 1056, 1064), ("wide", "bf16", 5950, 5120, 5128)])
def test_quantise_many_rows_bit_exact(cuda, kind, type, rows, K, ld):
    """Enough rows that CTAs walk several."""
    check_quantise(cuda, F4.NV, kind, type, rows, K, ld)


@pytest.mark.gpu
def test_rows_in_one_call_are_those_of_many_calls(cuda):
    """Many rows (walked by CTAs) against 2048 at a time (a CTA each), infinities and NaNs among them, bit for bit."""
    rows, K = 19000, 1056
    x = torch.randn(rows, K, device=cuda).bfloat16()
    x[::7] *= 2.0 ** -120
    x[5, 1055], x[4000, 0], x[18999, 7], x[130] = float("nan"), float("inf"), float("-inf"), 0
    codes, tiles, row = gpu_quantise(x, F4.NV)
    parts = [gpu_quantise(x[i:i + 2048], F4.NV) for i in range(0, rows, 2048)]
    for whole, n in ((codes, 0), (tiles, 1), (row, 2)):
        assert torch.equal(whole.view(torch.uint8), torch.cat([part[n] for part in parts]).view(torch.uint8))
    assert torch.isnan(row).nonzero().flatten().tolist() == [5, 4000, 18999]


def check_quantise(cuda, f, kind, type, rows, K, ld):
    dtype = TYPES[type][0]
    x = torch.from_numpy(rows_like(rows, ld, rows + K, kind)).clamp(-3e38, 3e38).to(dtype)
    x = x.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(cuda)
    spare = 64
    codes, tiles, row = gpu_quantise(x, f, K, spare)
    want_codes, want_bytes, want_row, q = F4.quantise(x[:, :K].double().cpu().numpy(), f)
    cb, sb = H.fp4_sizes(rows, K, f)
    packed, want_tiles = F4.pack(want_codes, want_bytes)
    assert (codes[cb:] == 0xEE).all() and (tiles[sb:] == 0xEE).all()
    np.testing.assert_array_equal(tiles[:sb].cpu().numpy(), want_tiles)  # the padding's zeros too
    if f == F4.NV:
        np.testing.assert_array_equal(row[:rows].cpu().numpy().astype(np.float64), want_row)
        assert (row[rows:] == -1).all()
    got, _ = F4.unpack(codes[:cb].cpu().numpy().reshape(rows, K // 2), want_tiles, f)
    got = np.where(got == 8, 0, got)  # a negative zero is a zero
    differ = got != want_codes
    if dtype == torch.float32 and f == F4.NV:
        # an fp32 quotient is rounded once (2^-24) before it is compared with the border between two codes
        borders = (F4.VALUES[1:] + F4.VALUES[:-1]) / 2
        near = (np.abs(np.abs(q)[..., None] - borders) <= 2.0 ** -23 * borders).any(-1)
        differ &= ~near
    assert not differ.any(), (np.argwhere(differ)[:5], got[differ][:5], want_codes[differ][:5], q[differ][:5])


@pytest.mark.gpu
@pytest.mark.parametrize("type,power", [("bf16", n) for n in (-126, -120, -118, -107, 0, 100, 116)] + [("f16", n) for n in (-12, 0, 4)])
def test_quantise_on_and_beside_every_border_of_every_scale(cuda, type, power):
    """Blocks of every e4m3 scale c with +-t c for the borders t between codes, exact and one step to either side; row scales 2^power."""
    dtype = TYPES[type][0]
    scales = [c for c in F4.e4m3_values().tolist() if 0 < c <= 320]
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    blocks = [np.concatenate([[6 * c], borders * c, -borders * c, [0.0]]) for c in scales]
    x = np.concatenate([[2047.0] + [1.0] * 15] + blocks + [np.zeros(16)] * ((len(blocks) + 1) % 2))
    x = torch.from_numpy(np.stack([x] * 3) * 2.0 ** power).to(dtype)
    bits = x.view(torch.int16)
    inner = torch.ones(x.shape[1], dtype=torch.bool)
    inner[::16] = False  # the blocks' largest stay
    inner &= x[0] != 0
    bits[1, inner] += 1
    bits[2, inner] -= 1
    got_codes, got_tiles, row = gpu_quantise(x.to(cuda), F4.NV)
    codes, bytes_, want_row, _ = F4.quantise(x.double().numpy(), F4.NV)
    packed, tiles = F4.pack(codes, bytes_)
    np.testing.assert_array_equal(got_tiles.cpu().numpy(), tiles)
    np.testing.assert_array_equal(row.cpu().numpy().astype(np.float64), want_row)
    got, _ = F4.unpack(got_codes.cpu().numpy().reshape(x.shape[0], -1), tiles, F4.NV)
    np.testing.assert_array_equal(np.where(got == 8, 0, got), codes)


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("type", list(TYPES))
def test_quantise_says_nan_where_the_input_is_not_finite(cuda, f, type):
    x = torch.ones(4, 128, dtype=TYPES[type][0], device=cuda)
    x[1, 40], x[2, 127], x[3, 0] = float("nan"), float("inf"), float("-inf")
    codes, tiles, row = gpu_quantise(x, f)
    want_codes, want_bytes, want_row, _ = F4.quantise(x.double().cpu().numpy(), f)
    packed, want_tiles = F4.pack(want_codes, want_bytes)
    np.testing.assert_array_equal(codes.cpu().numpy().reshape(4, 64), packed)
    np.testing.assert_array_equal(tiles.cpu().numpy(), want_tiles)
    if f == F4.NV:
        np.testing.assert_array_equal(row.cpu().numpy(), want_row.astype(np.float32))
    out = torch.zeros(4, 128, device=cuda)
    H.check(H.lib().h3k_dequant_rows_fp4(p(codes), p(tiles), p(row), 4, 128, f, H.F32, p(out), 128, stream()))
    sync()
    np.testing.assert_array_equal(out.cpu().numpy(), F4.values(want_codes, want_bytes, want_row if f == F4.NV else None, f).astype(np.float32))


@pytest.mark.gpu
def test_quantise_rows_that_share_their_memory(cuda):
    """ldx 0: every row is the same one (a broadcast input)."""
    x = torch.randn(64, device=cuda).bfloat16()
    rows = x.expand(5, 64)
    codes, tiles, row = gpu_quantise(rows, F4.NV)
    c = codes.view(5, 32)
    assert (c == c[0]).all() and (row == row[0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("rows,K,ldo", [(1, 32, 32), (131, 160, 168), (9, 5120, 5120)])
def test_dequantise_every_code_and_scale(cuda, f, type, rows, K, ldo):
    g = np.random.default_rng(K)
    codes = g.integers(0, 16, (rows, K), dtype=np.uint8)
    bytes_ = g.integers(0, 256 if f == F4.MX else 128, (rows, K // F4.BLOCK[f]), dtype=np.uint8)
    row = np.exp(g.standard_normal(rows)).astype(np.float32)
    packed, tiles = F4.pack(codes, bytes_)
    dtype, t = TYPES[type]
    out = torch.full((rows, ldo), 7.0, dtype=dtype, device=cuda)
    dp, dt, dr = (torch.from_numpy(np.ascontiguousarray(a)).to(cuda) for a in (packed, tiles, row))
    H.check(H.lib().h3k_dequant_rows_fp4(p(dp), p(dt), p(dr), rows, K, f, t, p(out), ldo, stream()))
    sync()
    with np.errstate(over="ignore"):
        exact = F4.values(codes, bytes_, None, f)
        want = torch.from_numpy((exact.astype(np.float32) * row[:, None]).astype(np.float32)).to(dtype)  # one fp32 product, one rounding
    assert (out[:, K:] == 7).all()
    got = out[:, :K].cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0, 0, 0), want.nan_to_num(0, 0, 0))


def operand(rows, K, f, seed, cuda, scale=1.0):
    """A 4-bit matrix on the GPU and its float64 values."""
    x = np.random.default_rng(seed).standard_normal((rows, K)) * scale
    codes, bytes_, row, _ = F4.quantise(x, f)
    packed, tiles = F4.pack(codes, bytes_)
    r = torch.from_numpy(row.astype(np.float32)).to(cuda) if f == F4.NV else None
    return torch.from_numpy(packed).to(cuda), torch.from_numpy(tiles).to(cuda), r, torch.from_numpy(F4.values(codes, bytes_, row, f)).to(cuda)


def product(A, B, f, epi, **kw):
    a = H.h3k_gemm_args(M=A[0].shape[0], N=B[0].shape[0], K=A[0].shape[1] * 2, a_scale=p(A[2]), b_scale=p(B[2]), eps=1e-6,
                        **{k: p(v) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    H.check(H.lib().h3k_gemm_fp4(p(A[0]), p(A[1]), p(B[0]), p(B[1]), f, ctypes.byref(a), epi, stream()))
    sync()


def bound(A, B):
    """How far an fp32 sum of the exact products may be off, whatever its order: each of the K additions by a step of 2^-23
    of a partial sum, which the sum of magnitudes bounds."""
    return A[3].shape[1] * 2.0 ** -23 * (A[3].abs() @ B[3].abs().T)


SHAPES = [(1, 8, 32), (1, 256, 64), (2, 264, 96), (127, 40, 160), (128, 256, 256), (129, 520, 288), (300, 768, 1024), (77, 512, 2080), (640, 1288, 5120), (5, 5120, 5120)]


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_f32_and_bf16(cuda, f, M, N, K):
    A, B = operand(M, K, f, M + K, cuda), operand(N, K, f, N + K + 1, cuda, 0.02)
    bias = torch.randn(N, device=cuda)
    want = A[3] @ B[3].T + bias.double()
    tol = bound(A, B) + 2.0 ** -22 * want.abs()  # the row scales' products and the bias, in fp32
    ldo = (N + 15) // 8 * 8
    out = torch.full((M + 1, ldo), 7.0, device=cuda)
    product(A, B, f, H.EPI_F32, out=out, ldo=ldo, bias=bias)
    assert ((out[:M, :N] - want).abs() <= tol).all(), ((out[:M, :N] - want).abs() / tol).max()
    assert (out[M] == 7).all() and (out[:, N:] == 7).all()
    low = torch.full((M + 1, ldo), 7.0, device=cuda, dtype=torch.bfloat16)
    product(A, B, f, H.EPI_BF16, out=low, ldo=ldo, bias=bias)
    assert ((low[:M, :N] - want).abs() <= tol + 2.0 ** -8 * want.abs()).all()
    assert (low[M] == 7).all() and (low[:, N:] == 7).all()


def sigmoid(x):
    return 1 / (1 + torch.exp(-x))


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("M,F,K", [(1, 128, 64), (130, 384, 256), (260, 4992, 1056)])
def test_product_swiglu(cuda, f, M, F, K):
    A, B = operand(M, K, f, M + K, cuda), operand(2 * F, K, f, F, cuda, 0.1)
    bias = torch.randn(2 * F, device=cuda) * 0.1
    y = A[3] @ B[3].T + bias.double()
    t = bound(A, B) + 2.0 ** -22 * y.abs()
    y, t = y.view(M, -1, 2, 128), t.view(M, -1, 2, 128)
    g, u, tg, tu = y[:, :, 0], y[:, :, 1], t[:, :, 0], t[:, :, 1]
    want = (g * sigmoid(g) * u).reshape(M, F)
    # |silu'| <= 1.1; the fp32 exponential, quotient and product: 2^-20 in all
    tol = (1.1 * tg * u.abs() + (g * sigmoid(g)).abs() * tu + tg * tu).reshape(M, F) + (2.0 ** -8 + 2.0 ** -20) * want.abs()
    out = torch.full((M + 1, F + 8), 7.0, device=cuda, dtype=torch.bfloat16)
    product(A, B, f, H.EPI_SWIGLU, out=out, ldo=F + 8, bias=bias)
    assert ((out[:M, :F] - want).abs() <= tol).all()
    assert (out[M] == 7).all() and (out[:, F:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 264, 96), (200, 640, 512)])
def test_product_gated_residual(cuda, f, M, N, K):
    A, B = operand(M, K, f, M, cuda), operand(N, K, f, N, cuda, 0.05)
    bias, mod = torch.randn(N, device=cuda), torch.randn(3, 6, N, device=cuda)
    idx = (torch.arange(M, device=cuda) % 3).to(torch.uint8)
    x = torch.randn(M + 1, N + 4, device=cuda)
    before = x.clone()
    product(A, B, f, H.EPI_GATE_RESID, x=x, ldx=N + 4, bias=bias, mod=mod, mod_idx=idx, gate_slot=5, dim=N)
    gate = mod[idx.long(), 5].double()
    y = A[3] @ B[3].T + bias.double()
    want = before[:M, :N].double() + gate * y
    tol = gate.abs() * (bound(A, B) + 2.0 ** -22 * y.abs()) + 2.0 ** -23 * (want.abs() + (gate * y).abs())
    assert ((x[:M, :N] - want).abs() <= tol).all()
    assert torch.equal(x[M], before[M]) and torch.equal(x[:, N:], before[:, N:])


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("M,heads,K,spare", [(1, 2, 64, 0), (300, 4, 512, 3)])
def test_product_qkv(cuda, f, M, heads, K, spare):
    inner = heads * 128
    A, B = operand(M, K, f, M, cuda), operand(3 * inner, K, f, K, cuda, 0.1)
    bias = torch.randn(3 * inner, device=cuda) * 0.1
    wq, wk = (1 + 0.1 * torch.randn(128, device=cuda) for _ in range(2))
    angle = torch.rand(M, 48, device=cuda, dtype=torch.float64) * 6.28
    rope = torch.stack([angle.cos(), angle.sin()], 2).float().contiguous()
    out = torch.full((M + spare, 3, heads, 128), 7.0, device=cuda, dtype=torch.bfloat16)
    product(A, B, f, H.EPI_QKV, out=out, bias=bias, rope=rope, qn_w=wq, kn_w=wk, inner=inner, heads_per_rank=heads, rows_local=M + spare)
    y = (A[3] @ B[3].T + bias.double()).view(M, 3, heads, 128)
    t = (bound(A, B) + 2.0 ** -22 * (A[3] @ B[3].T + bias.double()).abs()).view(M, 3, heads, 128)
    want, tol = y.clone(), t.clone()
    for sec, w in ((0, wq), (1, wk)):
        rms = (y[:, sec].square().mean(-1, keepdim=True) + 1e-6).sqrt()
        v = y[:, sec] / rms * w.double()
        c, s = rope[:, None, :, 0].double(), rope[:, None, :, 1].double()
        want[:, sec, :, :48], want[:, sec, :, 48:96], want[:, sec, :, 96:] = v[..., :48] * c - v[..., 48:96] * s, v[..., 48:96] * c + v[..., :48] * s, v[..., 96:]
        # a relative error of the row's norm is at most the largest of its elements' over the norm; a rotated element has
        # two terms
        e = t[:, sec] / rms * w.abs().double()
        e = 2 * e.amax(-1, keepdim=True) * (1 + v.abs()) + 2.0 ** -20 * v.abs().amax(-1, keepdim=True)
        tol[:, sec] = 2 * e
    tol = tol + 2.0 ** -8 * want.abs()
    assert ((out[:M] - want).abs() <= tol).all()
    assert (out[M:] == 7).all()  # the block's rows past M


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
def test_product_of_many_tiles_per_cta(cuda, f):
    """Every CTA works through both accumulators and the rings several times; rows sampled from every row tile."""
    M, N, K = 8263, 2056, 672
    g = torch.Generator(device="cpu").manual_seed(0)
    a = torch.randn(M, K, generator=g).bfloat16().to(cuda)
    b = torch.randn(N, K, generator=g).bfloat16().to(cuda)
    A, B = gpu_quantise(a, f), gpu_quantise(b, f)
    out = torch.zeros(M, N, device=cuda)
    args = H.h3k_gemm_args(M=M, N=N, K=K, a_scale=p(A[2]), b_scale=p(B[2]), out=p(out), ldo=N)
    H.check(H.lib().h3k_gemm_fp4(p(A[0]), p(A[1]), p(B[0]), p(B[1]), f, ctypes.byref(args), H.EPI_F32, stream()))
    sync()
    rows = np.unique(np.concatenate([np.arange(0, M, 61), [M - 1]]))
    va, vb = (torch.from_numpy(F4.values(*F4.unpack(t[0].view(n, -1).cpu().numpy(), t[1].cpu().numpy(), f), None if t[2] is None else t[2].cpu().numpy(), f)).to(cuda)
              for t, n in ((A, M), (B, N)))
    va = va[torch.from_numpy(rows).to(cuda)]
    want = va @ vb.T
    tol = K * 2.0 ** -23 * (va.abs() @ vb.abs().T) + 2.0 ** -22 * want.abs()
    assert ((out[torch.from_numpy(rows).to(cuda)] - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
def test_product_keeps_a_nan_to_its_row_and_ignores_what_lies_behind(cuda, f):
    """A NaN in row 3 of A shows in row 3 of the product and nowhere else; the buffers are followed by NaN patterns."""
    M, N, K = 9, 40, 96
    a = torch.randn(M, K, device=cuda).bfloat16()
    a[3, 17] = float("nan")
    b = torch.randn(N, K, device=cuda).bfloat16()
    A, B = (tuple(t if t is None else torch.cat([t, torch.full((4096,), 255, dtype=torch.uint8, device=cuda).view(t.dtype)]) for t in gpu_quantise(x, f)) for x in (a, b))
    out = torch.zeros(M, N, device=cuda)
    args = H.h3k_gemm_args(M=M, N=N, K=K, a_scale=p(A[2]), b_scale=p(B[2]), out=p(out), ldo=N)
    H.check(H.lib().h3k_gemm_fp4(p(A[0]), p(A[1]), p(B[0]), p(B[1]), f, ctypes.byref(args), H.EPI_F32, stream()))
    sync()
    bad = torch.isnan(out)
    assert bad[3].all() and not bad[torch.arange(M, device=cuda) != 3].any()


@pytest.mark.gpu
def test_calls_in_a_graph_and_on_another_stream_repeat_bit_for_bit(cuda):
    M, N, K, f = 200, 512, 512, F4.NV
    x, b = torch.randn(M, K, device=cuda).bfloat16(), torch.randn(N, K, device=cuda).bfloat16()
    B = gpu_quantise(b, f)
    codes, tiles = (torch.empty(n, dtype=torch.uint8, device=cuda) for n in H.fp4_sizes(M, K, f))
    row, out = torch.empty(M, device=cuda), torch.zeros(M, N, device=cuda, dtype=torch.bfloat16)
    args = H.h3k_gemm_args(M=M, N=N, K=K, a_scale=p(row), b_scale=p(B[2]), out=p(out), ldo=N)

    def calls():
        H.check(H.lib().h3k_quant_rows_fp4(p(x), H.BF16, K, M, K, f, p(codes), p(tiles), p(row), stream()))
        H.check(H.lib().h3k_gemm_fp4(p(codes), p(tiles), p(B[0]), p(B[1]), f, ctypes.byref(args), H.EPI_BF16, stream()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    side.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    x.mul_(-2)  # a power of two: the same codes with other signs, the same scales doubled
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, -2 * first)


# shapes by the form that the launch takes: K split over a cluster, CTAs that walk tiles of 128 rows, pairs of CTAs
FORMS = {"split": (77, 1288, 1056), "split rows": (257, 512, 800), "tiles": (100, 38408, 96), "one tile": (128, 256, 256), "pairs": (300, 7176, 352), "pair edge": (513, 6416, 544),
         "8 parts": (77, 1288, 3232), "8 parts of rows": (257, 512, 4000), "3 parts": (129, 5128, 10272), "3 parts, few rows": (20, 9480, 800),
         "2 parts, few rows": (31, 15368, 544), "pair of one": (128, 15368, 544)}


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("epilogue", ["bf16", "f32", "gate", "swiglu"])
def test_every_epilogue_in_every_form(cuda, f, form, epilogue):
    M, N, K = FORMS[form]
    if epilogue == "swiglu":
        N = (N + 255) // 256 * 256
    g = torch.Generator(device=cuda).manual_seed(M)
    A, B = (gpu_quantise((torch.randn(n, K, generator=g, device=cuda) * s).bfloat16(), f) for n, s in ((M, 1.0), (N, 0.1)))
    va, vb = (torch.from_numpy(F4.values(*F4.unpack(t[0].view(n, -1).cpu().numpy(), t[1].cpu().numpy(), f), None if t[2] is None else t[2].cpu().numpy(), f)).to(cuda)
              for t, n in ((A, M), (B, N)))
    bias = torch.randn(N, generator=g, device=cuda) * 0.1
    y = va @ vb.T + bias.double()
    t = K * 2.0 ** -23 * (va.abs() @ vb.abs().T) + 2.0 ** -22 * y.abs()
    A, B = ((x[0].view(n, -1), x[1], x[2]) for x, n in ((A, M), (B, N)))
    if epilogue == "gate":
        mod, idx = torch.randn(2, 6, N, generator=g, device=cuda), (torch.arange(M, device=cuda) % 2).to(torch.uint8)
        x = torch.randn(M + 1, N + 8, generator=g, device=cuda)
        before, gate = x.clone(), mod[idx.long(), 2].double()
        product(A, B, f, H.EPI_GATE_RESID, x=x, ldx=N + 8, bias=bias, mod=mod, mod_idx=idx, gate_slot=2, dim=N)
        want = before[:M, :N].double() + gate * y
        assert ((x[:M, :N] - want).abs() <= gate.abs() * t + 2.0 ** -23 * (want.abs() + (gate * y).abs())).all()
        assert torch.equal(x[M], before[M]) and torch.equal(x[:, N:], before[:, N:])
        return
    low = epilogue != "f32"
    if epilogue == "swiglu":
        y, t = y.view(M, -1, 2, 128), t.view(M, -1, 2, 128)
        gt, u, tg, tu = y[:, :, 0], y[:, :, 1], t[:, :, 0], t[:, :, 1]
        y = (gt * sigmoid(gt) * u).reshape(M, -1)
        t = (1.1 * tg * u.abs() + (gt * sigmoid(gt)).abs() * tu + tg * tu).reshape(M, -1) + 2.0 ** -20 * y.abs()
    n = y.shape[1]
    out = torch.full((M + 1, n + 8), 7.0, device=cuda, dtype=torch.bfloat16 if low else torch.float32)
    product(A, B, f, {"bf16": H.EPI_BF16, "f32": H.EPI_F32, "swiglu": H.EPI_SWIGLU}[epilogue], out=out, ldo=n + 8, bias=bias)
    assert ((out[:M, :n] - y).abs() <= t + (2.0 ** -8 * y.abs() if low else 0)).all()
    assert (out[M] == 7).all() and (out[:, n:] == 7).all()


@pytest.mark.gpu
def test_product_without_bias_or_row_scales_and_one_row_of_any_pitch(cuda):
    M, N, K, f = 1, 264, 544, F4.NV
    A, B = operand(M, K, f, 1, cuda), operand(N, K, f, 2, cuda)
    out = torch.full((N + 8,), 7.0, device=cuda)
    product((A[0], A[1], None), (B[0], B[1], None), f, H.EPI_F32, out=out, ldo=3)  # one row: no pitch
    want = (A[3] / A[2].double()[:, None]) @ (B[3] / B[2].double()[:, None]).T
    tol = K * 2.0 ** -23 * ((A[3] / A[2].double()[:, None]).abs() @ (B[3] / B[2].double()[:, None]).abs().T)
    assert ((out[:N] - want[0]).abs() <= tol[0]).all() and (out[N:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
def test_pairs_that_follow_one_another_at_once(cuda, f):
    """Products of one and of a few pairs of CTAs, whose clusters end while others start on the same SMs, queued on two streams without
    a wait: every result is bit for bit that of the call alone."""
    calls = []
    for M, N, K in ((128, 15368, 544), (300, 776, 352), (513, 264, 96), (130, 4104, 256)):
        A, B = operand(M, K, f, M, cuda), operand(N, K, f, N, cuda, 0.1)
        out = [torch.zeros(M, N, device=cuda, dtype=torch.bfloat16) for _ in range(2)]
        args = [H.h3k_gemm_args(M=M, N=N, K=K, a_scale=p(A[2]), b_scale=p(B[2]), out=p(o), ldo=N) for o in out]
        calls.append((A, B, out, args))
    go = lambda A, B, args: H.check(H.lib().h3k_gemm_fp4(p(A[0]), p(A[1]), p(B[0]), p(B[1]), f, ctypes.byref(args), H.EPI_BF16, stream()))
    want = []
    for A, B, out, args in calls:
        go(A, B, args[0])
        sync()
        want.append(out[0].clone())
    sides = [torch.cuda.Stream() for _ in range(2)]
    for i in range(200):
        for s, side in enumerate(sides):
            with torch.cuda.stream(side):
                A, B, out, args = calls[(i + 2 * s) % len(calls)]
                go(A, B, args[s])
    torch.cuda.synchronize()
    sync()
    for w, (A, B, out, args) in zip(want, calls):
        assert torch.equal(out[0], w) and torch.equal(out[1], w)


def test_sizes_whose_whole_tiles_leave_an_int_are_refused():
    """K, and a product's rows and columns, are rounded up to whole steps of up to 256."""
    L, most = H.lib(), 0x7fffff00
    assert H.fp4_sizes(1, most, F4.NV) == (most // 2, most // 64 * 512)
    for K in (most + 32, 0x7fffffe0):
        for f in FORMATS:
            refused(L.h3k_fp4_sizes(1, K, f, None, None), "K must be")
        refused(L.h3k_quant_rows_fp4(BASE, H.BF16, 0, 1, K, F4.MX, BASE, BASE, None, None), "K must be")
        refused(L.h3k_dequant_rows_fp4(BASE, BASE, None, 1, K, F4.MX, H.BF16, BASE, K, None), "K must be")
    for change, text in ((dict(M=most + 1), "rows"), (dict(N=most + 8), "columns"), (dict(K=most + 32), "K must be")):
        a = H.h3k_gemm_args(**(dict(M=1, N=256, K=64, out=BASE, ldo=0x7fffffff // 8 * 8) | change))
        refused(L.h3k_gemm_fp4(BASE, BASE, BASE, BASE, F4.MX, ctypes.byref(a), H.EPI_BF16, None), text)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K", [(3, 64), (3, 576), (300, 64)], ids=["one stage", "split", "pairs"])
def test_swiglu_of_gates_far_below_zero(cuda, M, K):
    """Gates from -80 to -88.5, whose sigmoids are down to 2^-127.7, with values that make up for them: bias alone sets both, the
    product is 0."""
    F = 128
    codes = lambda n: torch.zeros(n, K // 2, dtype=torch.uint8, device=cuda)
    tiles = lambda n: torch.zeros(H.fp4_sizes(n, K, F4.MX)[1], dtype=torch.uint8, device=cuda)
    gate, up = torch.linspace(-80, -88.5, F, device=cuda), torch.exp2(torch.linspace(100, 126, F, device=cuda))
    bias = torch.cat([gate, up])
    out = torch.zeros(M, F, device=cuda, dtype=torch.bfloat16)
    product((codes(M), tiles(M), None), (codes(2 * F), tiles(2 * F), None), F4.MX, H.EPI_SWIGLU, out=out, ldo=F, bias=bias)
    g = gate.double()
    want = g * sigmoid(g) * up.double()
    # fp32: the exponential of a number near 88 is off by its argument's rounding in base 2 (128 x 2^-24) and 2 ulp; sum, quotient (2 ulp)
    # and products by 2^-21 in all; then one rounding to bf16
    assert ((out - want).abs() <= (2.0 ** -8 + 2.0 ** -15) * want.abs()).all(), ((out - want).abs() / want.abs()).max()


def check_exactly(x, cuda):
    """NV codes, scales and row scales of fp32 rows, bit for bit, ties included."""
    got_codes, got_tiles, row = gpu_quantise(x.to(cuda), F4.NV)
    codes, bytes_, want_row, _ = F4.quantise(x.double().numpy(), F4.NV)
    packed, tiles = F4.pack(codes, bytes_)
    np.testing.assert_array_equal(got_tiles.cpu().numpy(), tiles)
    np.testing.assert_array_equal(row.cpu().numpy().astype(np.float64), want_row)
    got, _ = F4.unpack(got_codes.cpu().numpy().reshape(x.shape[0], -1), tiles, F4.NV)
    np.testing.assert_array_equal(np.where(got == 8, 0, got), codes)


@pytest.mark.gpu
@pytest.mark.parametrize("power", [-126, -120, -118, -107, -30, 0, 100, 116])
def test_quantise_fp32_on_and_beside_every_border_of_every_scale(cuda, power):
    """As above for fp32, up to four steps to either side. (x has 24 bits and t c at most seven, so an x beside the border is
    more than half a step of the quotient from it: one correct rounding does not reach it.)"""
    scales = [c for c in F4.e4m3_values().tolist() if 0 < c <= 320]
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    blocks = [np.concatenate([[6 * c], borders * c, -borders * c, [0.0]]) for c in scales]
    x = np.concatenate([[2047.0] + [1.0] * 15] + blocks + [np.zeros(16)] * ((len(blocks) + 1) % 2))
    x = torch.from_numpy(np.stack([x] * 9) * 2.0 ** power).float()
    bits = x.view(torch.int32)
    inner = torch.ones(x.shape[1], dtype=torch.bool)
    inner[::16] = False
    inner &= x[0] != 0
    for i, steps in enumerate((0, 1, -1, 2, -2, 3, -3, 4, -4)):
        bits[i, inner] += steps
    check_exactly(x, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "ties", "wide"])
@pytest.mark.parametrize("rows,K", [(1, 32), (130, 160), (33, 2048), (5, 4160), (7, 8224), (3, 40000)])
def test_quantise_fp32_exactly(cuda, kind, rows, K):
    check_exactly(torch.from_numpy(rows_like(rows, K, rows + K + 1, kind)).clamp(-3e38, 3e38).float(), cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("M,heads,per,K,spare", [(300, 8, 1, 96, 5), (129, 8, 4, 512, 0), (1, 16, 2, 64, 2), (100, 52, 52, 96, 0), (100, 52, 13, 96, 3), (128, 56, 7, 288, 1)])
def test_product_qkv_for_several_ranks(cuda, f, M, heads, per, K, spare):
    """Heads in groups of `per`, each with a block of its own behind the one before; pairs of CTAs, and at most 128 rows by many single
    ones. Rows behind M of every block stay as they are."""
    inner, ranks = heads * 128, heads // per
    A, B = operand(M, K, f, M, cuda), operand(3 * inner, K, f, K, cuda, 0.1)
    bias = torch.randn(3 * inner, device=cuda) * 0.1
    wq, wk = (1 + 0.1 * torch.randn(128, device=cuda) for _ in range(2))
    angle = torch.rand(M, 48, device=cuda, dtype=torch.float64) * 6.28
    rope = torch.stack([angle.cos(), angle.sin()], 2).float().contiguous()
    out = torch.full((ranks + 1, M + spare, 3, per, 128), 7.0, device=cuda, dtype=torch.bfloat16)
    product(A, B, f, H.EPI_QKV, out=out, bias=bias, rope=rope, qn_w=wq, kn_w=wk, inner=inner, heads_per_rank=per, rows_local=M + spare)
    y = (A[3] @ B[3].T + bias.double()).view(M, 3, heads, 128)
    t = (bound(A, B) + 2.0 ** -22 * (A[3] @ B[3].T + bias.double()).abs()).view(M, 3, heads, 128)
    want, tol = y.clone(), t.clone()
    c, s = rope[:, None, :, 0].double(), rope[:, None, :, 1].double()
    for sec, w in ((0, wq), (1, wk)):
        rms = (y[:, sec].square().mean(-1, keepdim=True) + 1e-6).sqrt()
        v = y[:, sec] / rms * w.double()
        want[:, sec, :, :48], want[:, sec, :, 48:96], want[:, sec, :, 96:] = v[..., :48] * c - v[..., 48:96] * s, v[..., 48:96] * c + v[..., :48] * s, v[..., 96:]
        e = t[:, sec] / rms * w.abs().double()
        tol[:, sec] = 2 * (2 * e.amax(-1, keepdim=True) * (1 + v.abs()) + 2.0 ** -20 * v.abs().amax(-1, keepdim=True))  # as in test_product_qkv
    tol = tol + 2.0 ** -8 * want.abs()
    got = out[:ranks, :M].permute(1, 2, 0, 3, 4).reshape(M, 3, heads, 128)  # [rank][row][3][slot] -> [row][3][head]
    assert ((got - want).abs() <= tol).all()
    assert (out[:ranks, M:] == 7).all() and (out[ranks] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f", FORMATS)
@pytest.mark.parametrize("K", [64, 1056], ids=["pair", "split"])
@pytest.mark.parametrize("N", [8, 264, 512])
def test_one_row_of_any_pitch_in_every_epilogue(cuda, f, K, N):
    """A single row has no pitch to check: ldo and ldx of 3."""
    A, B = operand(1, K, f, 1, cuda), operand(N, K, f, 2, cuda, 0.1)
    y = A[3] @ B[3].T
    t = bound(A, B) + 2.0 ** -22 * y.abs()
    for epi, dtype in ((H.EPI_F32, torch.float32), (H.EPI_BF16, torch.bfloat16)):
        out = torch.full((N + 8,), 7.0, device=cuda, dtype=dtype)
        product(A, B, f, epi, out=out, ldo=3)
        assert ((out[:N] - y[0]).abs() <= (t + (2.0 ** -8 * y.abs() if dtype == torch.bfloat16 else 0))[0]).all() and (out[N:] == 7).all()
    x, mod = torch.randn(N + 8, device=cuda), torch.randn(1, 6, N, device=cuda)
    before, idx = x.clone(), torch.zeros(1, dtype=torch.uint8, device=cuda)
    product(A, B, f, H.EPI_GATE_RESID, x=x, ldx=3, mod=mod, mod_idx=idx, gate_slot=1, dim=N)
    gate = mod[0, 1].double()
    want = before[:N].double() + gate * y[0]
    assert ((x[:N] - want).abs() <= gate.abs() * t[0] + 2.0 ** -23 * (want.abs() + (gate * y[0]).abs())).all() and torch.equal(x[N:], before[N:])
