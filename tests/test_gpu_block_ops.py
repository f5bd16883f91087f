"""RMS norm, linear with activation and differential attention (-m gpu) against plain implementations in 64 bits.

Tolerances.  u(t) = torch.finfo(t).eps / 2 is the largest relative error of one rounding to t (fp32: U = 2^-24).
  norm    |y - y64| <= (u + 3e-6) |y64| + tiny: the square sum has at most 72 additions in a row (64 elements a thread, 8 tree steps) for C <= 16384, i.e. 72 U
          relative, half of that after the root, and six single operations: (36 + 6) U < 3e-6; u is the final rounding, `tiny` half the type's smallest number.
  linear  accumulation: (K + 8) 2^-23 sum_k |x w| (one step per addition, whatever the order); the activations' slopes are at most 1.13; the activation functions
          themselves are within 2e-6 (1 + |v|); then one rounding u.  e4m3 operands with a 16-bit result: the matrix instruction keeps, of each 8 consecutive k, the
          products down to 2^-13 of the largest one's power of two, so a group of 8 loses less than 7 * 2^-13 max |x w| more.  (fp32 results do not use it.)
  attn    see attn_bound."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32, F8 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn
U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    from streamingt2v_amd import ops as o
    return o


def u(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps / 2      # half the smallest subnormal


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return lambda *s, scale=1.0: torch.randn(*s, generator=g, device="cuda") * scale


def within(name, got, want, bound):
    got, want, bound = got.double(), want.double(), bound.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    err = torch.where(torch.isnan(want) | (got == want), torch.zeros_like(want), (got - want).abs())
    worst = (err / bound.clamp_min(1e-300)).max().item() if err.numel() else 0.0
    print(f"[{name}] worst error / bound {worst:.3f}")
    assert worst <= 1.0, f"{name}: error {worst:.3f} times the bound"


# ------------------------------------------------------------------------------------------------------------- rmsnorm
def norm64(x, r, gamma, eps):
    s = x.double() + (r.double() if r is not None else 0)
    g = gamma.double() if gamma is not None else 1.0
    return s, s * g / (s.square().mean(1, keepdim=True) + eps).sqrt()


def check_norm(name, got, x, r, gamma, eps, f8):
    got = list(got) if isinstance(got, tuple) else [got]
    s, y = norm64(x, r, gamma, eps)
    if f8:
        q, a = got[0], got[1]
        a64 = y.abs().amax(1) / 448
        within(name + " scale", a, a64, (3e-6 + 2 * U32) * a64 + 1e-45)
        within(name + " values", q.double() * a.double()[:, None], y, (2.0 ** -4 + 5e-6) * y.abs() + 2.0 ** -10 * a64[:, None] + 1e-45)
        assert q.double().abs().amax(1)[a64 > 0].eq(448).all(), "each row's largest value stands at 448"
    else:
        t = got[0].dtype
        within(name, got[0], y, (u(t) + 3e-6) * y.abs() + tiny(t))
    if r is not None:
        t = got[-1].dtype
        within(name + " sum", got[-1], s, (u(t) + U32) * s.abs() + tiny(t))


NORM_SIZES = [(1, 1), (1, 5), (3, 7), (2, 8), (1, 1280), (5, 64), (33, 320), (129, 640), (7, 1277), (64, 1280), (3, 5120), (2, 10007), (1, 16384), (9, 2049), (300, 40)]


@pytest.mark.parametrize("f8", [False, True], ids=["e16", "e4m3"])
@pytest.mark.parametrize("xt,rt", [(F16, None), (BF16, None), (F32, None), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32), (F32, F32)], ids=str)
def test_rmsnorm_sizes(ops, xt, rt, f8):
    for i, (rows, ch) in enumerate(NORM_SIZES):
        randn = gen(100 + i)
        x = randn(rows, ch).to(xt)
        r = randn(rows, ch, scale=3.0).to(rt) if rt is not None else None
        gamma = 1 + randn(ch, scale=0.2) if i % 3 else None
        check_norm(f"rmsnorm {rows}x{ch} {xt} {rt}", ops.rmsnorm(x, gamma, eps=1e-6, residual=r, f8=f8), x, r, gamma, 1e-6, f8)


@pytest.mark.parametrize("pad,off", [(8, 0), (8, 8), (1, 0), (3, 1), (16, 4)])
@pytest.mark.parametrize("f8", [False, True], ids=["e16", "e4m3"])
def test_rmsnorm_strided_rows_and_destinations(ops, pad, off, f8):
    """Column ranges of wider buffers, at aligned and unaligned offsets; what lies around the destinations stays."""
    randn = gen(7)
    rows, ch = 19, 648
    wide = lambda t, fill: torch.full((rows, ch + pad + off), fill, device="cuda").to(t)  # noqa: E731
    x, r = wide(BF16, 0.0), wide(F32, 0.0)
    x[:, off:off + ch], r[:, off:off + ch] = randn(rows, ch).to(BF16), randn(rows, ch)
    xs, rs = x[:, off:off + ch], r[:, off:off + ch]
    out, osum = wide(F8 if f8 else BF16, 3.0), wide(F32, 5.0)
    gamma = 1 + randn(ch, scale=0.1)
    got = ops.rmsnorm(xs, gamma, residual=rs, f8=f8, out=out[:, off:off + ch], out_sum=osum[:, off:off + ch])
    assert got[0].data_ptr() == out[:, off:].data_ptr() and got[-1].data_ptr() == osum[:, off:].data_ptr()
    check_norm(f"rmsnorm strided pad {pad} off {off}", got, xs, rs, gamma, 1e-6, f8)
    for buf, fill in ((out, 3.0), (osum, 5.0)):
        keep = torch.ones(ch + pad + off, dtype=torch.bool, device="cuda")
        keep[off:off + ch] = False
        assert buf.float()[:, keep].eq(fill).all()


@pytest.mark.parametrize("rt", [BF16, F32], ids=str)
@pytest.mark.parametrize("ch", [640, 1277, 20000])
def test_rmsnorm_residual_in_place(ops, rt, ch):
    randn = gen(8)
    x, r = randn(37, ch).to(BF16), randn(37, ch).to(rt)
    before = r.clone()
    got = ops.rmsnorm(x, None, residual=r, out_sum=r)
    assert got[1].data_ptr() == r.data_ptr()
    check_norm("rmsnorm in place", got, x, before, None, 1e-6, False)


def test_rmsnorm_special_rows(ops):
    """A row of zeros, one with a NaN, one with an infinity, subnormals, the type's largest value."""
    x = gen(9)(6, 640).to(F16)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 639] = float("inf")
    x[3] = x[3] * 2.0 ** -20
    x[4, 7] = 65504
    q, a = ops.rmsnorm(x, None, f8=True)
    y = ops.rmsnorm(x, None)
    assert q[0].float().eq(0).all() and a[0].item() == 0 and y[0].eq(0).all()
    assert torch.isnan(q[1].float()).all() and torch.isnan(a[1]) and torch.isnan(y[1]).all()
    assert torch.isnan(q[2].float()).all() and torch.isnan(a[2]) and torch.isnan(y[2, 639])
    check_norm("rmsnorm special", (q[3:], a[3:]), x[3:], None, None, 1e-6, True)
    check_norm("rmsnorm special", y[3:], x[3:], None, None, 1e-6, False)


@pytest.mark.parametrize("xt", [F32, BF16], ids=str)
@pytest.mark.parametrize("ch", [64, 1277, 12000])
def test_rmsnorm_tiny_rows_in_8_bits(ops, xt, ch):
    """Rows so small that max |y| / 448 is below the smallest normal number: the scale stops there, and the values are numbers.
    |scale q - y| <= (2^-4 + 5e-6) |y| + 2^-10 scale, as for any row; y's own rounding below 2^-126 is 2^-150, far below 2^-10 2^-126."""
    randn = gen(23)
    x = torch.cat([randn(2, ch) * s for s in (1e-30, 1e-36, 1e-38, 1e-39)]).to(xt)
    gamma = 1 + randn(ch, scale=0.1)
    q, a = ops.rmsnorm(x, gamma, eps=1e-6, f8=True)
    _, y = norm64(x, None, gamma, 1e-6)
    a64 = (y.abs().amax(1) / 448).clamp_min(2.0 ** -126)
    within("rmsnorm tiny rows: scale", a, a64, (3e-6 + 2 * U32) * a64)
    within("rmsnorm tiny rows: values", q.double() * a.double()[:, None], y, (2.0 ** -4 + 5e-6) * y.abs() + 2.0 ** -10 * a64[:, None])


def test_rmsnorm_empty_and_many_rows(ops):
    assert ops.rmsnorm(torch.empty(0, 640, dtype=F16, device="cuda")).shape == (0, 640)
    q, a, s = ops.rmsnorm(torch.empty(0, 640, dtype=F16, device="cuda"), residual=torch.empty(0, 640, dtype=F32, device="cuda"), f8=True)
    assert q.shape == (0, 640) and a.shape == (0,) and s.dtype == F32
    x = gen(10)(70001, 24).to(BF16)
    check_norm("rmsnorm 70001 rows", ops.rmsnorm(x, None), x, None, None, 1e-6, False)


def test_rmsnorm_more_threads_than_a_launch_has(ops):
    """2^28 rows of 16 threads each would be 2^32: another form takes them."""
    rows = (1 << 28) + 5
    x = torch.empty(rows, 8, dtype=F16, device="cuda")
    at = [slice(0, 1000), slice(rows // 2, rows // 2 + 1000), slice(rows - 1000, rows)]
    for i, a in enumerate(at):
        x[a] = gen(40 + i)(1000, 8).to(F16)
    y = ops.rmsnorm(x, None)
    for a in at:
        check_norm("rmsnorm 2^28 rows", y[a], x[a], None, None, 1e-6, False)


# ---------------------------------------------------------------------------------------------------------- linear_act
ACTS = {None: lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh"),
        "silu": torch.nn.functional.silu}


def quant(t):
    a = t.abs().amax(1) / 448
    return (t / a[:, None]).to(F8), a


def make_linear(seed, m, n, k, t):
    randn = gen(seed)
    x, w = randn(m, k), randn(n, k, scale=k ** -0.5)
    if t == F8:
        (x, sx), (w, sw) = quant(x), quant(w)
        return randn, x, w, sx, sw
    return randn, x.to(t), w.to(t), None, None


def group_max(x, w):
    """sum over groups of 8 consecutive k of the group's largest x[m, k] w[n, k]."""
    pad = -x.shape[1] % 8
    x, w = (torch.nn.functional.pad(a.float(), (0, pad)).unflatten(1, (-1, 8)) for a in (x, w))
    out = torch.zeros(x.shape[0], w.shape[0], device="cuda")
    for g in range(x.shape[1]):
        top = x[:, None, g, 0] * w[None, :, g, 0]
        for j in range(1, 8):
            top = torch.maximum(top, x[:, None, g, j] * w[None, :, g, j])
        out += top
    return out.double() * 1.001


def check_linear(name, got, x, w, sx, sw, bias, act, res):
    xd, wd = x.double(), w.double()
    if sx is not None:
        xd = xd * sx.double()[:, None]
    if sw is not None:
        wd = wd * sw.double()[:, None]
    v = xd @ wd.t()
    b = (x.shape[1] + 8) * 2.0 ** -23 * (xd.abs() @ wd.abs().t()) + 3 * U32 * v.abs()
    if x.dtype == F8 and got.dtype != F32:
        b = b + 7 * 2.0 ** -13 * group_max(xd.abs(), wd.abs())
    if bias is not None:
        v = v + bias.double()
        b = b + U32 * v.abs()
    want = ACTS[act](v)
    b = 1.13 * b + (2e-6 * (1 + v.abs()) if act in ("gelu", "gelu_tanh", "silu") else 0)
    if res is not None:
        want = want + res.double()
    t = got.dtype
    within(name, got, want, b + (u(t) + 2 * U32) * (want.abs() + b) + tiny(t))


LIN_SIZES = [(1, 1, 1), (1, 64, 64), (2, 33, 17), (5, 1001, 515), (31, 96, 640), (33, 130, 72), (77, 320, 1024), (64, 64, 4096), (128, 128, 128), (129, 257, 130),
             (200, 640, 320), (300, 1280, 48), (513, 300, 264), (1, 5120, 1280), (16, 1280, 5120), (257, 513, 1040)]


@pytest.mark.parametrize("t", [F16, BF16, F8], ids=str)
def test_linear_sizes(ops, t):
    for i, (m, n, k) in enumerate(LIN_SIZES):
        randn, x, w, sx, sw = make_linear(200 + i, m, n, k, t)
        act = list(ACTS)[i % 5]
        e = F16 if t == F8 and i % 2 else BF16 if t == F8 else t
        od = F32 if i % 4 == 1 else e
        bias = randn(n, scale=0.3) if i % 3 else None
        res = randn(m, n).to([e, F32][i % 2]) if i % 4 != 2 else None
        got = ops.linear_act(x, w, bias=bias, act=act, residual=res, x_scale=sx, w_scale=sw, out_dtype=od)
        check_linear(f"linear {m}x{n}x{k} {t} {act}", got, x, w, sx, sw, bias, act, res)


FEW_ROWS = [(1, 1280, 5120), (8, 1280, 2560), (9, 1280, 2560), (16, 2560, 320), (17, 2560, 320), (3, 9, 5117), (8, 2048, 64), (5, 321, 63), (1, 2049, 65), (16, 4096, 1029), (64, 512, 4096), (33, 100, 129)]


@pytest.mark.parametrize("t", [F16, BF16, F8], ids=str)
def test_linear_few_rows(ops, t):
    """Every number of columns to a workgroup, and K shorter and longer than what its waves take at once; a NaN in one row or column stays there."""
    for i, (m, n, k) in enumerate(FEW_ROWS):
        randn, x, w, sx, sw = make_linear(260 + i, m, n, k, t)
        e = BF16 if t == F8 else t
        for od in (e, F32):
            got = ops.linear_act(x, w, act="silu", x_scale=sx, w_scale=sw, out_dtype=od)
            check_linear(f"linear {m}x{n}x{k} {t} {od}", got, x, w, sx, sw, None, "silu", None)
        x2, w2 = x.clone(), w.clone()
        x2.view(torch.uint8)[m // 2].fill_(0x7f)          # NaN in e4m3 and bf16, fp16 (0x7f7f)
        w2.view(torch.uint8)[n // 3].fill_(0x7f)
        bad = ops.linear_act(x2, w2, act="silu", x_scale=sx, w_scale=sw, out_dtype=e)
        same = ops.linear_act(x, w, act="silu", x_scale=sx, w_scale=sw, out_dtype=e)
        keep = torch.ones(m, n, dtype=torch.bool, device="cuda")
        keep[m // 2], keep[:, n // 3] = False, False
        assert torch.equal(bad[keep], same[keep])


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("t", [F16, F8], ids=str)
def test_linear_activations_reach_far_values(ops, act, t):
    """The activation's whole range: a product of a diagonal puts -40 .. 40 (and the borders around 0) on every output."""
    n = 160
    x = torch.eye(n, device="cuda").to(t)
    w = torch.linspace(-40, 40, n * n, device="cuda").reshape(n, n)
    w[0] = 0.0
    w = w.to(t)
    got = ops.linear_act(x, w, act=act, out_dtype=F32)
    check_linear(f"linear act {act}", got, x, w, None, None, None, act, None)


@pytest.mark.parametrize("t", [F16, BF16, F8], ids=str)
@pytest.mark.parametrize("m,n,k", [(3, 272, 208), (70, 272, 208), (300, 272, 208), (1100, 1040, 208), (1100, 1041, 209), (1100, 1040, 80), (4100, 2064, 208), (4100, 2064, 64), (4096, 2048, 320), (1100, 1040, 2064),
                                   (8448, 2176, 1120)])
def test_linear_picks_rows_and_columns(ops, t, m, n, k):
    """One-hot rows select columns of W: any swapped lane, row or K chunk shows as another number, exactly.  Few rows, 128- and 256-row tiles, unaligned rows, one to
    many K steps with and without a rest."""
    x = torch.zeros(m, k, device="cuda")
    idx = (torch.arange(m, device="cuda") * 7) % k
    x[torch.arange(m, device="cuda"), idx] = 1
    w = ((torch.arange(n * k, device="cuda") * 37) % 61 - 30).reshape(n, k).to(t) if t != F8 else ((torch.arange(n * k, device="cuda") * 37) % 31 - 15).reshape(n, k).float().to(t)
    got = ops.linear_act(x.to(t), w, out_dtype=F32)
    assert torch.equal(got, w.float().t()[idx])


@pytest.mark.parametrize("t", [BF16, F8], ids=str)
@pytest.mark.parametrize("m,n,k", [(3, 320, 640), (90, 320, 640), (600, 328, 640), (1200, 1040, 640)])
@pytest.mark.parametrize("off", [0, 16, 3])
def test_linear_views_and_in_place_residual(ops, t, m, n, k, off):
    """Operands and destination are column ranges of wider rows; the destination is the residual; what surrounds it stays."""
    randn, x, w, sx, sw = make_linear(11, m, n, k, t)
    xb = torch.full((m, k + 2 * 16), float("nan"), device="cuda").to(t)
    wb = torch.full((n, k + 2 * 16), float("nan"), device="cuda").to(t)
    xb[:, off:off + k], wb[:, off:off + k] = x, w
    yb = torch.full((m, n + 2 * 16), 9.0, device="cuda").to(BF16)
    res = randn(m, n).to(BF16)
    y = yb[:, off:off + n]
    y.copy_(res)
    got = ops.linear_act(xb[:, off:off + k], wb[:, off:off + k], act="relu", residual=y, x_scale=sx, w_scale=sw, out=y)
    assert got.data_ptr() == y.data_ptr()
    check_linear("linear views", got, x, w, sx, sw, None, "relu", res)
    assert yb[:, :off].float().eq(9).all() and yb[:, off + n:].float().eq(9).all()


@pytest.mark.parametrize("t", [F16, F8], ids=str)
def test_linear_rows_do_not_mix(ops, t):
    """A NaN row stays in its row, an Inf weight row in its column; empty input."""
    for m in (5, 200):
        randn, x, w, sx, sw = make_linear(12, m, 160, 320, t)
        x[2] = float("nan")
        w[7] = float("nan")
        got = ops.linear_act(x, w, act="relu", x_scale=sx, w_scale=sw, out_dtype=F32)
        nan = torch.isnan(got)
        assert nan[2].all() and nan[:, 7].all() and nan.sum().item() == m + 160 - 1
    assert ops.linear_act(x[:0], w, x_scale=sx[:0] if sx is not None else None, w_scale=sw).shape == (0, 160)


@pytest.mark.parametrize("t", [BF16, F8], ids=str)
def test_linear_product_sizes(ops, t):
    for i, (m, n, k) in enumerate([(2304, 5120, 1280), (2304, 1280, 5120), (4096, 3840, 1280), (1000, 2560, 640), (3000, 2998, 1296), (1111, 1501, 333)]):
        randn, x, w, sx, sw = make_linear(300 + i, m, n, k, t)
        bias, res = randn(n), randn(m, n).to(F32 if i % 2 else BF16)
        got = ops.linear_act(x, w, bias=bias, act="gelu", residual=res, x_scale=sx, w_scale=sw, out_dtype=res.dtype)
        part = torch.arange(0, m, 37, device="cuda")          # every row of every tile is covered by test_linear_picks_rows_and_columns
        check_linear(f"linear {m}x{n}x{k} {t}", got[part], x.float()[part].to(t), w, sx[part] if sx is not None else None, sw, bias, "gelu", res[part])


# ----------------------------------------------------------------------------------------------------------- attn_diff
def visible(B, n_q, n_k, causal, k_len, q_start):
    n = k_len.long().clamp(0, n_k) if k_len is not None else torch.full((B,), n_k, device="cuda")
    last = n[:, None].expand(B, n_q)
    if causal:
        first = q_start.long() if q_start is not None else n - n_q
        last = torch.minimum(last, first[:, None] + torch.arange(1, n_q + 1, device="cuda"))
    return torch.arange(n_k, device="cuda")[None, None] < last[..., None]              # [B, n_q, n_k]


def attn64(q, k, v, lam, lam_init, gamma, eps, causal, k_len, q_start):
    """(result, bound).  Every weight of a map is rounded to the 16-bit type once (u, or half the smallest number of fp16 below its normals, relative to a row maximum of 1 whose sum is
    at least 1); a score's error d changes a weight by d: 70 products and additions of at most |q| |k| / 8, and the exponential's argument and result; every
    tile of keys rescales once.  So each map's product is off by at most (u + d) A|V| + n tiny max|V|.  The head norm scales that by 1 / rms and adds the change of rms."""
    B, n_q, H, _ = q.shape
    n_k, KV = k.shape[1], k.shape[2]
    see = visible(B, n_q, n_k, causal, k_len, q_start)
    l = lam.double()
    lamv = ((l[0] * l[1]).sum().exp() - (l[2] * l[3]).sum().exp() + lam_init).item()
    out = torch.zeros(B, n_q, H, 128, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    t = q.dtype
    for h in range(H):
        kh = h // (H // KV)
        vv = torch.nan_to_num(v[:, :, kh].double(), nan=0.0, posinf=0.0, neginf=0.0)
        o, b = 0.0, 0.0
        for i, f in ((0, 1.0), (1, -lamv)):
            qq, kk = q[:, :, h, 64 * i:64 * i + 64].double(), torch.nan_to_num(k[:, :, kh, 64 * i:64 * i + 64].double(), nan=0.0)
            s = (qq @ kk.transpose(1, 2).contiguous()) / 8
            a = torch.softmax(s.masked_fill(~see, -math.inf), -1)
            a = torch.where(see, a, torch.zeros_like(a))
            d = 70 * U32 * (qq.abs() @ kk.abs().transpose(1, 2).contiguous()).amax().item() / 8 + 8 * U32 + (n_k / 32 + 8) * U32 * 2
            o = o + f * (a @ vv)
            b = b + abs(f) * ((u(t) + 2 * d) * (a @ vv.abs()) + n_k * tiny(t) * vv.abs().max().item())
        if gamma is not None:
            rms = (o.square().mean(-1, keepdim=True) + eps).sqrt()
            g = gamma.double().abs() * (1 - lam_init)
            b = g / rms * (b + o.abs() / rms * b.square().mean(-1, keepdim=True).sqrt())
            o = o * gamma.double() * (1 - lam_init) / rms
        out[:, :, h], bound[:, :, h] = o, b + (u(t) + 8 * U32) * (o.abs() + b) + tiny(t)
    return out, bound


def run_attn(ops, name, q, k, v, seed, layer=2, norm=True, causal=False, k_len=None, q_start=None, out=None, k_ref=None, v_ref=None):
    randn = gen(seed + 5000)
    lam, lam_init = randn(4, 64, scale=0.1), 0.8 - 0.6 * math.exp(-0.3 * layer)
    gamma = 1 + randn(128, scale=0.1) if norm else None
    got = ops.attn_diff(q, k, v, lam, lam_init, gamma=gamma, causal=causal, k_len=k_len, q_start=q_start, out=out)
    want, bound = attn64(q, k if k_ref is None else k_ref, v if v_ref is None else v_ref, lam, lam_init, gamma, 1e-5, causal, k_len, q_start)
    within(name, got, want, bound)
    return got


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


ATTN_SIZES = [(1, 1, 1, 1, 1), (2, 1, 33, 2, 1), (1, 3, 64, 4, 4), (3, 25, 25, 2, 2), (2, 77, 77, 4, 2), (1, 130, 257, 3, 3), (2, 33, 1000, 8, 1), (1, 1, 1025, 8, 8),
              (4, 1, 700, 16, 2), (1, 2, 4099, 5, 5), (2, 31, 32, 2, 2), (1, 32, 31, 2, 2), (1, 64, 65, 6, 2), (1, 300, 64, 2, 1), (40, 9, 9, 2, 2), (2, 5, 129, 7, 1)]


@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
@pytest.mark.parametrize("t", [F16, BF16], ids=str)
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
def test_attn_sizes(ops, t, causal, norm):
    for i, (B, n_q, n_k, H, KV) in enumerate(ATTN_SIZES):
        randn = gen(400 + i)
        q, k, v = randn(B, n_q, H, 128).to(t), randn(B, n_k, KV, 128).to(t), randn(B, n_k, KV, 128).to(t)
        run_attn(ops, f"attn {B} {n_q}x{n_k} {H}/{KV} {t}", q, k, v, i, layer=i % 6, norm=norm, causal=causal)


@pytest.mark.parametrize("t", [F16, BF16], ids=str)
@pytest.mark.parametrize("n_q,n_k,H,KV", [(1, 500, 4, 2), (40, 500, 4, 2), (300, 300, 2, 2)])
def test_attn_lengths_and_what_lies_behind_them(ops, t, n_q, n_k, H, KV):
    """Lengths of 0, 1, a tile's border and all; the cache behind a sequence's last key holds NaN and Inf; lengths out of range are clamped."""
    lens = [0, 1, 31, 32, 33, 64, n_k - 1, n_k, n_k + 7, -3]
    B = len(lens)
    randn = gen(500)
    q, k, v = randn(B, n_q, H, 128).to(t), randn(B, n_k, KV, 128).to(t), randn(B, n_k, KV, 128).to(t)
    k_bad, v_bad = k.clone(), v.clone()
    for b, n in enumerate(lens):
        k_bad[b, max(n, 0):], v_bad[b, max(n, 0):] = float("nan"), float("inf")
    for causal, start in ((False, None), (True, None), (True, ints(*[5 * b for b in range(B)]))):
        got = run_attn(ops, f"attn lengths causal {causal}", q, k_bad, v_bad, 1, causal=causal, k_len=ints(*lens), q_start=start, k_ref=k, v_ref=v)
        assert got[0].eq(0).all() and got[-1].eq(0).all()


def test_attn_causal_positions(ops):
    """Queries in front of the first key, inside, and far behind the last (positions that pass 31 bits with the query added)."""
    randn = gen(501)
    B, n_q, n_k = 6, 50, 120
    q, k, v = randn(B, n_q, 4, 128).to(BF16), randn(B, n_k, 2, 128).to(BF16), randn(B, n_k, 2, 128).to(BF16)
    start = ints(-60, -20, 0, 37, 110, 2 ** 31 - 5)
    got = run_attn(ops, "attn positions", q, k, v, 2, causal=True, q_start=start)
    assert got[0].eq(0).all() and got[1, :20].eq(0).all()


@pytest.mark.parametrize("t", [F16, BF16], ids=str)
@pytest.mark.parametrize("n", [40, 200])
def test_attn_what_a_query_does_not_see_does_not_reach_it(ops, t, n):
    """Causal: NaN or Inf in keys and values of a position reach the queries from that position on and no earlier one, in the same tile or another."""
    randn = gen(502)
    q, k, v = randn(1, n, 2, 128).to(t), randn(1, n, 2, 128).to(t), randn(1, n, 2, 128).to(t)
    lam = torch.zeros(4, 64, device="cuda")
    want, bound = attn64(q, k, v, lam, 0.4, None, 1e-5, True, None, None)
    for at in (1, 5, 31, 32, 39, n - 1):
        for bad in ("nan", "inf"):
            k2, v2 = k.clone(), v.clone()
            v2[0, at, :, 3] = float(bad)
            k2[0, at, :, 7] = float("nan")
            got = ops.attn_diff(q, k2, v2, lam, 0.4, causal=True)
            within(f"attn in front of a {bad} at {at}", got[:, :at], want[:, :at], bound[:, :at])
            assert torch.isnan(got[:, at:]).any(-1).all()


@pytest.mark.parametrize("t", [F16, BF16], ids=str)
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("B,n_q,n_k,H,KV", [(1, 1, 256, 8, 8), (2, 1, 255, 16, 1), (1, 16, 256, 2, 2), (3, 4, 129, 8, 2), (1, 1, 66, 1, 1), (5, 2, 200, 8, 1), (4, 1, 257, 4, 4), (3, 17, 250, 2, 2)])
def test_attn_short_caches(ops, t, B, n_q, n_k, H, KV, causal):
    """A few rows on up to 256 keys, lengths from none to all, whatever lies in what is not seen, and the largest scores in one wave's keys only."""
    randn = gen(503)
    q, k, v = randn(B, n_q, H, 128).to(t), randn(B, n_k, KV, 128).to(t), randn(B, n_k, KV, 128).to(t)
    k[:, 40:44] *= 8
    lens = [n_k, 0, 1, n_k // 2, 33][:B]
    k2, v2 = k.clone(), v.clone()
    for b, n in enumerate(lens):
        k2[b, n:], v2[b, n:] = float("nan"), float("inf")
    run_attn(ops, f"attn short caches {B} {n_q}x{n_k} {H}/{KV} {t}", q, k2, v2, 7, causal=causal, k_len=ints(*lens), k_ref=k, v_ref=v)
    if causal:          # something not finite that only later queries see
        lam = torch.zeros(4, 64, device="cuda")
        want, bound = attn64(q, k, v, lam, 0.4, None, 1e-5, True, None, None)
        v[:, n_k - 1] = float("nan")
        got = ops.attn_diff(q, k, v, lam, 0.4, causal=True)
        within("attn short caches: a NaN at the end", got[:, :-1], want[:, :-1], bound[:, :-1])
        assert torch.isnan(got[:, -1]).all()


@pytest.mark.parametrize("n_q", [1, 25, 150])
def test_attn_views(ops, n_q):
    """Column ranges of a fused projection; (frame, pixel) rows; [batch, kv head, capacity, 128] caches; a strided destination whose surroundings stay."""
    randn = gen(503)
    B, H, KV = 6, 4, 2
    rows = randn(B, n_q, (H + 2 * KV) * 128).to(F16)
    q, k, v = (x.unflatten(2, (-1, 128)) for x in rows.split([H * 128, KV * 128, KV * 128], 2))
    run_attn(ops, "attn fused rows", q, k, v, 3)
    buf = torch.full((B, n_q + 3, H + 1, 128), 7.0, dtype=F16, device="cuda")
    got = run_attn(ops, "attn strided destination", q, k, v, 3, out=buf[:, 1:n_q + 1, :H])
    assert got.data_ptr() == buf[:, 1:].data_ptr()
    assert buf[:, 0].eq(7).all() and buf[:, n_q + 1:].eq(7).all() and buf[:, :, H].eq(7).all()
    rows = randn(n_q, B, (H + 2 * KV) * 128).to(F16)
    q, k, v = (x.unflatten(2, (-1, 128)).transpose(0, 1) for x in rows.split([H * 128, KV * 128, KV * 128], 2))
    run_attn(ops, "attn frame rows", q, k, v, 4)
    kc, vc = randn(B, KV, 333, 128).to(F16), randn(B, KV, 333, 128).to(F16)
    run_attn(ops, "attn head-major cache", q, kc.transpose(1, 2), vc.transpose(1, 2), 5, k_len=ints(333, 1, 200, 64, 0, 17))


def test_attn_large_and_equal_scores(ops):
    """Scores far apart (one key takes all), all equal, growing along the keys (every tile raises the maximum), and at fp16's limits of the weights."""
    randn = gen(504)
    B, n_q, n_k, H = 1, 40, 900, 1
    q, v = randn(B, n_q, H, 128), randn(B, n_k, H, 128).to(F16)
    for name, k in (("equal", torch.zeros(B, n_k, H, 128, device="cuda")), ("growing", torch.linspace(0, 8, n_k, device="cuda")[None, :, None, None] * torch.sign(q[:, :1])),
                    ("one key", randn(B, n_k, H, 128) * (torch.arange(n_k, device="cuda") == 700)[None, :, None, None] * 12)):
        for t in (F16, BF16):
            run_attn(ops, "attn scores " + name, q.to(t), k.to(t), v.to(t), 6, norm=False)


@pytest.mark.parametrize("B,n_q,n_k,H,KV", [(3, 1, 600, 4, 2), (3, 3, 20, 4, 2), (80, 70, 90, 4, 2)])
def test_attn_zeros_stay_zeros_without_eps(ops, B, n_q, n_k, H, KV):
    """eps = 0: neither a query that sees no key nor one that sees only values of zero divides by zero; the others are as ever."""
    randn = gen(60)
    q, k, v = randn(B, n_q, H, 128).to(F16), randn(B, n_k, KV, 128).to(F16), randn(B, n_k, KV, 128).to(F16)
    v[1] = 0
    lens = torch.full((B,), n_k, dtype=torch.int32, device="cuda")
    lens[0] = 0
    lam, gamma = randn(4, 64, scale=0.1), 1 + randn(128, scale=0.1)
    got = ops.attn_diff(q, k, v, lam, 0.4, gamma=gamma, eps=0.0, k_len=lens)
    assert got[:2].eq(0).all()
    near = ops.attn_diff(q, k, v, lam, 0.4, gamma=gamma, eps=1e-12, k_len=lens)
    assert got[2:].ne(0).any() and torch.allclose(got[2:].float(), near[2:].float(), rtol=2.0 ** -9, atol=2.0 ** -24)          # a step of the type


def test_attn_empty(ops):
    lam = torch.zeros(4, 64, device="cuda")
    e = lambda *s: torch.empty(*s, dtype=F16, device="cuda")  # noqa: E731
    assert ops.attn_diff(e(0, 3, 2, 128), e(0, 5, 2, 128), e(0, 5, 2, 128), lam, 0.2).shape == (0, 3, 2, 128)
    assert ops.attn_diff(e(2, 0, 2, 128), e(2, 5, 2, 128), e(2, 5, 2, 128), lam, 0.2).shape == (2, 0, 2, 128)
    assert ops.attn_diff(e(2, 3, 2, 128), e(2, 0, 2, 128), e(2, 0, 2, 128), lam, 0.2).eq(0).all()


def test_attn_long_cache_offsets(ops):
    """A cache whose later rows lie behind 2^32 bytes of its start."""
    n_k, KV = 140000, 128
    k = torch.empty(1, n_k, KV, 128, dtype=BF16, device="cuda")
    v = torch.empty(1, n_k, KV, 128, dtype=BF16, device="cuda")
    assert k.numel() * 2 > 2 ** 32
    randn = gen(505)
    for h in (0, KV - 1):
        k[:, :, h], v[:, :, h] = randn(1, n_k, 128).to(BF16), randn(1, n_k, 128).to(BF16)
    q = randn(1, 1, 2, 128).to(BF16)
    run_attn(ops, "attn long cache", q, k[:, :, ::KV - 1], v[:, :, ::KV - 1], 7)


# ------------------------------------------------------------------------------------------------------------- together
def block(ops, x, stream, P, k_len, q_start):
    """One pre-norm block on x's rows with 8-bit products: norm -> q | k | v -> differential attention -> projection onto the stream -> norm -> feed-forward."""
    B, n, C = stream.shape
    H = P["heads"]
    t = {}
    t["n1"] = ops.rmsnorm(x, P["g1"], residual=stream.view(B * n, C), f8=True)
    t["qkv"] = ops.linear_act(t["n1"][0], P["wqkv"][0], x_scale=t["n1"][1], w_scale=P["wqkv"][1], out_dtype=BF16)
    q, k, v = (a.unflatten(2, (-1, 128)) for a in t["qkv"].view(B, n, -1).split([H * 128] * 3, 2))
    t["o"] = ops.attn_diff(q, k, v, P["lam"], 0.5, gamma=P["gh"], causal=True, k_len=k_len, q_start=q_start)
    t["x1"] = ops.linear_act(t["o"].view(B * n, -1), P["wo"], bias=P["bo"], residual=t["n1"][2])
    t["n2"] = ops.rmsnorm(t["x1"], P["g2"], f8=True)
    t["h"] = ops.linear_act(t["n2"][0], P["w1"][0], bias=P["b1"], act="silu", x_scale=t["n2"][1], w_scale=P["w1"][1], out_dtype=BF16)
    t["y"] = ops.linear_act(t["h"], P["w2"], residual=t["x1"])
    return t


def block_params(C, H, F_):
    randn = gen(600)
    return dict(heads=H, g1=1 + randn(C, scale=0.1), g2=1 + randn(C, scale=0.1), gh=1 + randn(128, scale=0.1), lam=randn(4, 64, scale=0.1),
                wqkv=quant(randn(3 * H * 128, C, scale=C ** -0.5)), wo=randn(C, H * 128, scale=(H * 128) ** -0.5).to(BF16), bo=randn(C, scale=0.1),
                w1=quant(randn(F_, C, scale=C ** -0.5)), b1=randn(F_, scale=0.1), w2=randn(C, F_, scale=F_ ** -0.5).to(BF16))


@pytest.mark.parametrize("n", [1, 77, 300])
def test_block_run_together(ops, n):
    """Every stage of the run against 64 bits on the stage's own inputs: the stages' bounds hold as they stand."""
    B, C, H, F_ = 3, 640, 5, 1280
    P = block_params(C, H, F_)
    randn = gen(601 + n)
    x, stream = randn(B * n, C).to(BF16), randn(B, n, C).to(BF16)
    k_len, q_start = ints(n, max(n - 13, 1), 1), ints(0, 0, 0)
    t = block(ops, x, stream, P, k_len, q_start)
    check_norm("block n1", t["n1"], x, stream.view(B * n, C), P["g1"], 1e-6, True)
    check_linear("block qkv", t["qkv"], t["n1"][0], P["wqkv"][0], t["n1"][1], P["wqkv"][1], None, None, None)
    q, k, v = (a.unflatten(2, (-1, 128)) for a in t["qkv"].view(B, n, -1).split([H * 128] * 3, 2))
    want, bound = attn64(q, k, v, P["lam"], 0.5, P["gh"], 1e-5, True, k_len, q_start)
    within("block attention", t["o"], want, bound)
    check_linear("block x1", t["x1"], t["o"].view(B * n, -1), P["wo"], None, None, P["bo"], None, t["n1"][2])
    check_norm("block n2", t["n2"], t["x1"], None, P["g2"], 1e-6, True)
    check_linear("block h", t["h"], t["n2"][0], P["w1"][0], t["n2"][1], P["w1"][1], P["b1"], "silu", None)
    check_linear("block y", t["y"], t["h"], P["w2"], None, None, None, None, t["x1"])


@pytest.mark.parametrize("n", [1, 300])
def test_block_prompt_then_single_tokens(ops, n):
    """A prompt's keys and values go into a cache, single tokens follow: their attention equals that of the whole sequence at the same rows, within both bounds."""
    B, H, KV, cap = 2, 4, 2, n + 70
    randn = gen(602)
    q, k, v = randn(B, cap, H, 128).to(BF16), randn(B, cap, KV, 128).to(BF16), randn(B, cap, KV, 128).to(BF16)
    lam, gamma = randn(4, 64, scale=0.1), 1 + randn(128, scale=0.1)
    whole = ops.attn_diff(q, k, v, lam, 0.3, gamma=gamma, causal=True)
    _, bound = attn64(q, k, v, lam, 0.3, gamma, 1e-5, True, None, None)
    kc, vc = torch.full_like(k, float("nan")), torch.full_like(v, float("nan"))
    kc[:, :n], vc[:, :n] = k[:, :n], v[:, :n]
    for at in range(n, cap, 23):
        kc[:, n:at + 1], vc[:, n:at + 1] = k[:, n:at + 1], v[:, n:at + 1]
        one = ops.attn_diff(q[:, at:at + 1], kc, vc, lam, 0.3, gamma=gamma, k_len=ints(*[at + 1] * B))
        within(f"token {at}", one, whole[:, at:at + 1].double(), 2 * bound[:, at:at + 1])


def test_block_captured_and_replayed_between_eager_runs(ops):
    """Two graphs of the block (a prompt's and a single token's) replayed in turn, with eager runs and new inputs in between: every replay is the eager result, bit for bit."""
    B, C, H, F_ = 2, 640, 5, 1280
    P = block_params(C, H, F_)
    sizes = (150, 1)
    state = []
    for n in sizes:
        randn = gen(610 + n)
        x, stream, k_len, q_start = randn(B * n, C).to(BF16), randn(B, n, C).to(BF16), ints(n, n), ints(0, 0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(ops, x, stream, P, k_len, q_start)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            t = block(ops, x, stream, P, k_len, q_start)
        state.append((g, t, x, stream, k_len, q_start))
    for rep in range(4):
        for g, t, x, stream, k_len, q_start in state:
            randn = gen(620 + rep)
            x.copy_(randn(*x.shape))
            stream.copy_(randn(*stream.shape))
            eager = block(ops, x, stream, P, k_len, q_start)["y"].clone()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(t["y"], eager)
    kq = gen(630)
    q, k, v = kq(1, 1, 4, 128).to(BF16), kq(1, 9000, 4, 128).to(BF16), kq(1, 9000, 4, 128).to(BF16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ops.attn_diff(q, k, v, P["lam"], 0.5)
    for rep in range(3):
        q.copy_(kq(1, 1, 4, 128))
        eager = ops.attn_diff(q, k, v, P["lam"], 0.5).clone()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, eager)


def test_block_ops_on_two_streams_at_once(ops):
    """The same operators on two streams with different inputs, many times: scratch memory and results do not mix, and repeat bit for bit."""
    randn = gen(640)
    lam = randn(4, 64, scale=0.1)
    data, want = [], []
    for s in range(2):
        q, k, v = randn(2, 1, 8, 128).to(F16), randn(2, 6000, 4, 128).to(F16), randn(2, 6000, 4, 128).to(F16)
        x, w = randn(64, 1280).to(F16), randn(640, 1280, scale=0.03).to(F16)
        data.append((q, k, v, x, w))
        want.append((ops.attn_diff(q, k, v, lam, 0.4), ops.linear_act(x, w, act="gelu"), *ops.rmsnorm(x, f8=True)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                q, k, v, x, w = data[s]
                got[s].append((ops.attn_diff(q, k, v, lam, 0.4), ops.linear_act(x, w, act="gelu"), *ops.rmsnorm(x, f8=True)))
    torch.cuda.synchronize()
    for s in range(2):
        for g in got[s]:
            for a, b in zip(g, want[s]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
