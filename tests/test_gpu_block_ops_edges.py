"""RMS norm, linear with activation and differential attention at the ends of the numbers' range (-m gpu), against plain implementations in 64 bits.

Bounds: those of test_gpu_block_ops (U32 = 2^-24 is one fp32 rounding, u(t) one rounding to t, tiny(t) half the type's smallest number) unless a test derives its own."""
import math

import pytest
import torch

from tests.test_gpu_block_ops import ACTS, BF16, F16, F32, F8, U32, check_linear, check_norm, gen, make_linear, ops, run_attn, tiny, u, within  # noqa: F401

pytestmark = pytest.mark.gpu

NORM_WIDTHS = [5, 64, 640, 1277, 2560, 10007, 12000]          # 16, 64 and 256 threads to a row, aligned and not, and the one-row form


# ------------------------------------------------------------------------------------------------------------- rmsnorm
@pytest.mark.parametrize("f8", [False, True], ids=["e16", "e4m3"])
@pytest.mark.parametrize("xt,rt", [(F16, None), (BF16, BF16), (F32, None), (BF16, F32), (F32, F32)], ids=str)
def test_rmsnorm_rows_of_zeros_without_eps(ops, xt, rt, f8):
    """eps = 0: a row of zeros stays zeros (e4m3: with scale 0), the rows beside it are as ever."""
    for i, ch in enumerate(NORM_WIDTHS):
        randn = gen(900 + i)
        x, r = randn(6, ch).to(xt), randn(6, ch).to(rt) if rt is not None else None
        gamma = 1 + randn(ch, scale=0.1) if i % 2 else None
        for t in (x, r):
            if t is not None:
                t[1], t[4] = 0, 0
        got = ops.rmsnorm(x, gamma, eps=0.0, residual=r, f8=f8)
        got = list(got) if isinstance(got, tuple) else [got]
        for g in got:
            assert g[1].float().eq(0).all() and g[4].float().eq(0).all(), ch
        rest = [0, 2, 3, 5]
        check_norm(f"rmsnorm eps 0 {ch} {xt} {rt}", tuple(g[rest] for g in got), x[rest], r[rest] if r is not None else None, gamma, 0.0, f8)


@pytest.mark.parametrize("f8", [False, True], ids=["e16", "e4m3"])
@pytest.mark.parametrize("eps", [0.0, 1e-30])
def test_rmsnorm_rows_whose_squares_leave_fp32(ops, eps, f8):
    """Rows of 1e-38 to 1e37, and one with values of both ends: the result is the formula's, within the bounds of any row."""
    for i, ch in enumerate(NORM_WIDTHS):
        for xt, rt in ((F32, None), (BF16, None), (F32, F32), (BF16, F32)):
            randn = gen(920 + i)
            size = torch.tensor([1e-38, 1e-30, 1e-25, 1e-20, 1.0, 1e18, 1e20, 1e30, 1e37], device="cuda")[:, None]
            x = (randn(9, ch).clamp(-8, 8) * size).to(xt)
            x[4, 0], x[4, 1] = 1e30, 1e-30
            r = (randn(9, ch).clamp(-8, 8) * size).to(rt) if rt is not None else None
            gamma = 1 + randn(ch, scale=0.1) if i % 2 else None
            check_norm(f"rmsnorm squares out of range {ch} {xt} {rt}", ops.rmsnorm(x, gamma, eps=eps, residual=r, f8=f8), x, r, gamma, eps, f8)


@pytest.mark.parametrize("f8", [False, True], ids=["e16", "e4m3"])
def test_rmsnorm_fp32_rows_with_a_16_bit_residual(ops, f8):
    """fp32 x on a residual of the package's 16-bit type: the sum goes on in 16 bits, in place too."""
    for i, ch in enumerate(NORM_WIDTHS):
        randn = gen(930 + i)
        x, r = randn(7, ch), randn(7, ch, scale=3.0).to(ops.ELEM)
        gamma = 1 + randn(ch, scale=0.1) if i % 2 else None
        check_norm(f"rmsnorm fp32 + 16 bit {ch}", ops.rmsnorm(x, gamma, residual=r, f8=f8), x, r, gamma, 1e-6, f8)
        before = r.clone()
        check_norm(f"rmsnorm fp32 + 16 bit {ch} in place", ops.rmsnorm(x, gamma, residual=r, out_sum=r, f8=f8), x, before, gamma, 1e-6, f8)


# ---------------------------------------------------------------------------------------------------------- linear_act
FAR = [0.0, -0.0, 1e-30, -1e-30, 1.0, -1.0, 6.99, -6.99, 7.0, -7.0, 7.01, -7.01, 50.0, -50.0, 1e4, -1e4, 1e7, -1e7, 1e9, -1e9, 1e12, -1e12, 1e30, -1e30, 3e38, -3e38]


@pytest.mark.parametrize("t", [F16, BF16, F8], ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 300, 64), (40, 300, 700), (300, 1040, 128), (300, 1041, 128), (1100, 1040, 2064), (1101, 1041, 2067), (4400, 2100, 64)])
def test_linear_gelu_far_out(ops, t, m, n, k):
    """x = 0, so the bias alone is the activation's argument, to both ends of fp32 and beyond.  gelu is within 2e-6 of x Phi(x) over the whole range, and one rounding; +inf gives
    +inf, -inf the limit 0, NaN NaN."""
    x, w = torch.zeros(m, k, device="cuda").to(t), gen(940)(n, k).to(t)
    bias = torch.tensor(FAR, device="cuda").repeat(-(-n // len(FAR)))[:n].contiguous()
    bias[n - 1], bias[n // 2], bias[n // 3] = float("inf"), float("-inf"), float("nan")
    want = 0.5 * bias.double() * torch.erfc(-bias.double() / math.sqrt(2.0))
    want[n // 2] = 0.0
    for od in (F32, BF16 if t == F8 else t):
        got = ops.linear_act(x, w, bias=bias, act="gelu", out_dtype=od)
        same = torch.nan_to_num(got.float(), nan=0.125, posinf=0.375, neginf=-0.375)
        assert torch.equal(same, same[:1].expand(m, n)), "every row is the same"
        fits = want.abs() < torch.finfo(od).max          # (an fp16 result overflows to infinity behind 65504)
        fits[n - 1] = fits[n // 3] = True
        bound = 2e-6 + (u(od) + U32) * torch.nan_to_num(want.abs(), posinf=0.0) + tiny(od)
        within(f"gelu far out {m}x{n}x{k} {t} {od}", got[0][fits], want[fits], bound[fits])


def test_gelu_rows_far_out(ops):
    """The row pass on every finite 16-bit number and the infinities: within 2e-6 and one rounding of x Phi(x)."""
    for t in (F16, BF16):
        x = torch.arange(65536, device="cuda").to(torch.int32).to(torch.int16).view(t).reshape(256, 256)
        nan, inf = torch.isnan(x), torch.isinf(x)
        xd = x.double()
        want = torch.where(inf, xd.clamp_min(0), 0.5 * xd * torch.erfc(-xd / math.sqrt(2.0)))
        got = ops.gelu_(x.clone())
        bound = 2e-6 + (u(t) + U32) * torch.nan_to_num(want.abs(), nan=0.0, posinf=0.0) + tiny(t)
        within(f"gelu rows {t}", got, torch.where(nan, xd, want), bound)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", [(1, 300, 64), (300, 1041, 128), (1100, 1040, 2064), (4400, 2100, 64)])
def test_linear_activations_far_out(ops, act, m, n, k):
    """As for gelu: the other activations from the bias alone, to both ends of fp32, the infinities and NaN: 2e-6, and four roundings of a large result."""
    x, w = torch.zeros(m, k, device="cuda").to(BF16), gen(941)(n, k).to(BF16)
    bias = torch.tensor(FAR, device="cuda").repeat(-(-n // len(FAR)))[:n].contiguous()
    bias[n - 1], bias[n // 2], bias[n // 3] = float("inf"), float("-inf"), float("nan")
    want = ACTS[act](bias.double())
    for od in (F32, BF16):
        got = ops.linear_act(x, w, bias=bias, act=act, out_dtype=od)
        within(f"{act} far out {m}x{n}x{k} {od}", got[-1], want, 2e-6 + (u(od) + 4 * U32) * torch.nan_to_num(want.abs(), nan=0.0, posinf=0.0) + tiny(od))


@pytest.mark.parametrize("t", [BF16, F8], ids=str)
def test_linear_far_rows(ops, t):
    """Rows 2^23 bytes and more apart (tiles copy them), and rows of more than 2^23 bytes (few of them)."""
    es = 1 if t == F8 else 2
    ld = (1 << 23) // es + 16
    randn, x, w, sx, sw = make_linear(880, 1100, 1040, 320, t)
    far = torch.zeros(1100, ld * es, dtype=torch.uint8, device="cuda").view(t)[:, 8:328]
    far.view(torch.uint8).copy_(x.view(torch.uint8))
    check_linear("linear far rows", ops.linear_act(far, w, x_scale=sx, w_scale=sw, act="silu", out_dtype=BF16), x, w, sx, sw, None, "silu", None)
    del far
    k = (1 << 23) // es + 37
    randn, x, w, sx, sw = make_linear(881, 3, 5, k, t)
    got = ops.linear_act(x, w, x_scale=sx, w_scale=sw, out_dtype=F32)
    scale = sx.double()[:, None] * sw.double()[None] if sx is not None else 1.0
    # all ones in front of it: whole numbers below 2^24 are exact, so a piece of K that is left out or counted twice shows as another number
    one = torch.ones(3, k, device="cuda").to(t)
    assert ops.linear_act(one, one[:2], out_dtype=F32).eq(k).all()
    within("linear long rows", got, (x.double() @ w.double().t()) * scale, (k + 8) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t()) * scale)


# ----------------------------------------------------------------------------------------------------------- attn_diff
# wave form with one share, with shares and a join, one workgroup, many rows
ATTN_FORMS = [(600, 1, 4, 2, 300), (1, 1, 8, 8, 4099), (2, 3, 8, 2, 250), (16, 200, 4, 4, 1000)]


def heads_of(t, B, n, H):
    """[128] channel values in every row of [B, n, H, 128]."""
    return t.to("cuda")[None, None, None].expand(B, n, H, 128).contiguous()


@pytest.mark.parametrize("B,n_q,H,KV,n_k", ATTN_FORMS)
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_attn_small_weights_beside_a_large_one(ops, B, n_q, H, KV, n_k, norm):
    """fp16: one key of value 0 takes almost everything, the other keys' weights are 2^-26 of it, and they alone make the result.
    A weight stands at least 2^7 times as high as relative to the row's largest, so it is rounded by u, or below fp16's normals by 2^-25 / 2^7: each map is off by at most
    (u + d) A|V| + n_k 2^-32 max|V|, d as in test_gpu_block_ops.attn64; A's own difference follows."""
    randn = gen(960)
    step = torch.full((128,), 1.0)
    q = heads_of(step, B, n_q, H).to(F16)
    k = randn(B, n_k, KV, 128, scale=0.02).to(F16)
    k[:, 0] = 2.25          # 64 * 2.25 / 8 = 18, and 18 log2(e) = 25.97
    v = (64 + randn(B, n_k, KV, 128, scale=8.0)).to(F16)
    v[:, 0] = 0
    lam, lam_init = torch.zeros(4, 64, device="cuda"), 0.4
    gamma = 1 + randn(128, scale=0.1) if norm else None
    got = ops.attn_diff(q, k, v, lam, lam_init, gamma=gamma, eps=1e-12)
    want, bound = torch.zeros(B, n_q, H, 128, dtype=torch.float64, device="cuda"), None
    bound = torch.zeros_like(want)
    d = 70 * U32 * 64 * 2.25 / 8 + 8 * U32 + (n_k / 32 + 8) * U32 * 2
    for h in range(H):
        kh = h // (H // KV)
        o, b = 0.0, 0.0
        for i, f in ((0, 1.0), (1, -lam_init)):
            s = q[:, :1, h, 64 * i:64 * i + 64].double() @ k[:, :, kh, 64 * i:64 * i + 64].double().transpose(1, 2).contiguous() / 8          # all queries are the same
            a = torch.softmax(s, -1)
            o = o + f * (a @ v[:, :, kh].double())
            b = b + abs(f) * ((u(F16) + 2 * d) * (a @ v[:, :, kh].double().abs()) + n_k * 2.0 ** -32 * v[:, :, kh].double().abs().max().item())
        if norm:
            rms = (o.square().mean(-1, keepdim=True) + 1e-12).sqrt()
            g = gamma.double().abs() * (1 - lam_init)
            b = g / rms * (b + o.abs() / rms * b.square().mean(-1, keepdim=True).sqrt())
            o = o * gamma.double() * (1 - lam_init) / rms
        want[:, :, h], bound[:, :, h] = o, b + (u(F16) + 8 * U32) * (o.abs() + b) + tiny(F16)
    within(f"attn small weights {B} {n_q}x{n_k} {H}/{KV}", got, want, bound)


@pytest.mark.parametrize("t", [F16, BF16], ids=str)
@pytest.mark.parametrize("B,n_q,H,KV,n_k", ATTN_FORMS)
def test_attn_scores_of_minus_infinity_are_not_an_empty_row(ops, t, B, n_q, H, KV, n_k):
    """Every score of the rows that see a key is -inf (an infinity in each key): no softmax exists, the result is NaN, as for any infinity; a row that sees no key is zeros."""
    randn = gen(970)
    q, k, v = randn(B, n_q, H, 128).to(t), randn(B, n_k, KV, 128).to(t), randn(B, n_k, KV, 128).to(t)
    q[..., 0], q[..., 64] = 1.0, 1.0
    for at in (0, 64):          # in one map, then in the other
        k2 = k.clone()
        k2[..., at] = float("-inf")
        lens = torch.full((B,), n_k, dtype=torch.int32, device="cuda")
        lens[-1] = 0 if B > 1 else n_k
        got = ops.attn_diff(q, k2, v, torch.zeros(4, 64, device="cuda"), 0.4, k_len=lens)
        assert torch.isnan(got[:B - (B > 1)]).all()
        assert B == 1 or got[-1].eq(0).all()


@pytest.mark.parametrize("B,n_q,H,KV,n_k", ATTN_FORMS)
def test_attn_head_norm_of_values_whose_squares_leave_fp32(ops, B, n_q, H, KV, n_k):
    """bf16 values of 1e-30 (with eps = 0) to 1e30: the head's norm is the formula's.  With eps = 0 the result of values times 2^c is that of the values:
    the products and sums scale exactly, and the norm's factor is rounded anew (8 U32) in front of the result's rounding (both results': 2 u)."""
    randn = gen(980)
    q, k, v = randn(B, n_q, H, 128).to(BF16), randn(B, n_k, KV, 128).to(BF16), randn(B, n_k, KV, 128).to(BF16)
    lam, gamma = randn(4, 64, scale=0.1), 1 + randn(128, scale=0.1)
    want = ops.attn_diff(q, k, v, lam, 0.4, gamma=gamma, eps=0.0)
    for c in (-90, -70, 70, 100):
        got = ops.attn_diff(q, k, (v.float() * 2.0 ** c).to(BF16), lam, 0.4, gamma=gamma, eps=0.0)
        within(f"attn head norm 2^{c} {B} {n_q}x{n_k}", got, want, (u(BF16) * 2 + 8 * U32) * want.double().abs() + tiny(BF16))


@pytest.mark.parametrize("t", [F16, BF16], ids=str)
@pytest.mark.parametrize("B,n_q,H,KV,n_k", [(600, 1, 4, 2, 100), (2, 1, 8, 4, 3000), (3, 4, 8, 2, 200), (40, 200, 4, 4, 300)])
def test_attn_shared_prefix_views(ops, t, B, n_q, H, KV, n_k):
    """One cache for the whole batch (a batch stride of 0), one head's keys for every head (a head stride of 0), the same queries for every sequence; queries updated in place."""
    randn = gen(990)
    k, v = randn(1, n_k, KV, 128).to(t).expand(B, n_k, KV, 128), randn(1, n_k, 1, 128).to(t).expand(B, n_k, KV, 128)
    q = randn(1, n_q, H, 128).to(t).expand(B, n_q, H, 128)
    got = run_attn(ops, "attn shared prefix", q, k, v, 1, causal=n_q > 1)
    assert torch.equal(got, got[:1].expand_as(got).contiguous())
    q = randn(B, n_q, H, 128).to(t)
    want = run_attn(ops, "attn shared prefix, queries of their own", q, k, v, 2, causal=n_q > 1)
    randn = gen(5002)
    lam, lam_init = randn(4, 64, scale=0.1), 0.8 - 0.6 * math.exp(-0.6)
    got = ops.attn_diff(q, k, v, lam, lam_init, gamma=1 + randn(128, scale=0.1), causal=n_q > 1, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(q, want), "in place of the queries"
