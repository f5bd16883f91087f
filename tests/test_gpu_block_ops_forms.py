"""The forms of attn_diff and linear_act that a large call takes (-m gpu), against plain implementations in 64 bits: many query rows (rings of key and value tiles, the two maps in
turn), the last round of product tiles split over K and joined, and unaligned operands together with that split.  Bounds: those of test_gpu_block_ops."""
import pytest
import torch

from streamingt2v_amd.lib import DTYPE_BF16, DTYPE_F16, DTYPE_F8, LIN_OUT_F32, lib
from tests.test_gpu_block_ops import BF16, F16, F32, F8, attn64, check_linear, gen, ints, make_linear, ops, run_attn, within  # noqa: F401

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------------------------------------- attn_diff
def many_rows(B, n_q, n_k, H, KV):
    """Asserts that this call takes the form for many rows, which needs no scratch memory.  With over 16 rows on over 64 keys the other one needs some wherever it has fewer than 1024
    units of 32 rows, so there the scratch size tells; more blocks of 128 rows than in such a case take the same form."""
    rows = n_q * (H // KV)
    units, blocks = -(-rows // 32) * B * KV, -(-rows // 128) * B * KV
    assert rows > 64 and blocks >= 128 and n_k > 64 and lib.svd_attn_diff_ws_bytes(B, n_q, n_k, H, KV) == 0
    return units < 1024


#            blocks: 160, 150, 256, 288 (told apart by scratch memory), 576 (over 512: long rows first)
MANY_ROWS = [(16, 300, 300, 4, 2), (25, 100, 257, 6, 6), (64, 129, 513, 2, 2), (24, 300, 70, 4, 4), (8, 450, 450, 18, 18)]


def test_attn_many_rows_is_the_form_that_runs():
    assert [many_rows(*c) for c in MANY_ROWS] == [True, True, True, True, False]


@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
@pytest.mark.parametrize("t", [F16, BF16], ids=str)
@pytest.mark.parametrize("causal", [False, True], ids=["all", "causal"])
@pytest.mark.parametrize("size", MANY_ROWS, ids=str)
def test_attn_many_rows(ops, size, causal, t, norm):
    B, n_q, n_k, H, KV = size
    many_rows(*size)
    randn = gen(700 + B)
    q, k, v = randn(B, n_q, H, 128).to(t), randn(B, n_k, KV, 128).to(t), randn(B, n_k, KV, 128).to(t)
    run_attn(ops, f"attn many rows {size} {t}", q, k, v, B, norm=norm, causal=causal)


@pytest.mark.parametrize("t", [F16, BF16], ids=str)
@pytest.mark.parametrize("n_q,n_k,H,KV", [(300, 300, 4, 2), (70, 500, 8, 4), (129, 161, 10, 10)])
def test_attn_many_rows_lengths_and_positions(ops, t, n_q, n_k, H, KV):
    """Lengths from none to all and around the steps of 32, starts in front of, inside and behind the keys; what lies behind a length is NaN and Inf."""
    lens = [0, 1, 31, 32, 33, 63, 64, 65, 96, 97, 128, 129, n_k - 1, n_k, n_k + 7, -3, 5, 40, 100, n_k, n_k - 2, 127, n_k, n_k - 32, 160, 159]
    B = len(lens)
    many_rows(B, n_q, n_k, H, KV)
    randn = gen(720)
    q, k, v = randn(B, n_q, H, 128).to(t), randn(B, n_k, KV, 128).to(t), randn(B, n_k, KV, 128).to(t)
    k_bad, v_bad = k.clone(), v.clone()
    for b, n in enumerate(lens):
        k_bad[b, max(n, 0):], v_bad[b, max(n, 0):] = float("nan"), float("inf")
    starts = [0, -n_q, -40, 7, 2 ** 31 - 5, -1, 30, 64, n_k, 3, -100, 31, 33, 1, 0, 0, -2, 90, 17, n_k - n_q, 5, -64, -33, 96, 2, 1]
    for causal, start in ((False, None), (True, None), (True, ints(*starts))):
        got = run_attn(ops, f"attn many rows: lengths, causal {causal}", q, k_bad, v_bad, 1, causal=causal, k_len=ints(*lens), q_start=start, k_ref=k, v_ref=v)
        assert got[0].eq(0).all() and got[15].eq(0).all()


@pytest.mark.parametrize("t", [F16, BF16], ids=str)
def test_attn_many_rows_what_a_query_does_not_see_does_not_reach_it(ops, t):
    """Causal: NaN or Inf in a key and value reach the queries from that position on and no earlier one: the block starts over without them."""
    B, n, H = 32, 200, 2
    many_rows(B, n, n, H, H)
    randn = gen(730)
    q, k, v = randn(B, n, H, 128).to(t), randn(B, n, H, 128).to(t), randn(B, n, H, 128).to(t)
    lam = torch.zeros(4, 64, device="cuda")
    want, bound = attn64(q, k, v, lam, 0.4, None, 1e-5, True, None, None)
    clean = ops.attn_diff(q, k, v, lam, 0.4, causal=True)
    for bad in ("nan", "inf"):
        at = [(37 * b + 1) % n for b in range(B)]          # another position in every sequence
        at[:6] = [0, 31, 32, 127, 128, n - 1]
        k2, v2 = k.clone(), v.clone()
        for b in range(0, B, 2):          # every other sequence, and of those every head
            v2[b, at[b], :, 3] = float(bad)
            k2[b, at[b], :, 7] = float("nan")
        got = ops.attn_diff(q, k2, v2, lam, 0.4, causal=True)
        for b in range(0, B, 2):
            if at[b]:
                within(f"attn many rows: in front of a {bad} at {at[b]}", got[b, :at[b]], want[b, :at[b]], bound[b, :at[b]])
            assert torch.isnan(got[b, at[b]:]).any(-1).all()
        assert torch.equal(got[1::2], clean[1::2])


@pytest.mark.parametrize("t", [F16, BF16], ids=str)
def test_attn_many_rows_views_and_destinations(ops, t):
    """Column ranges of a projection's rows, (frame, pixel) rows, a head-major cache, a strided destination whose surroundings stay."""
    randn = gen(740)
    B, n, H, KV = 20, 140, 8, 4
    many_rows(B, n, n, H, KV)
    rows = randn(B, n, (H + 2 * KV) * 128).to(t)
    q, k, v = (x.unflatten(2, (-1, 128)) for x in rows.split([H * 128, KV * 128, KV * 128], 2))
    buf = torch.full((B, n + 3, H + 1, 128), 7.0, dtype=t, device="cuda")
    run_attn(ops, "attn many rows: views", q, k, v, 3, causal=True, out=buf[:, 1:n + 1, :H])
    assert buf[:, 0].eq(7).all() and buf[:, n + 1:].eq(7).all() and buf[:, :, H].eq(7).all()
    rows = randn(n, B, (H + 2 * KV) * 128).to(t)
    q, k, v = (x.unflatten(2, (-1, 128)).transpose(0, 1) for x in rows.split([H * 128, KV * 128, KV * 128], 2))
    run_attn(ops, "attn many rows: frame rows", q, k, v, 4)
    kc, vc = randn(B, KV, 333, 128).to(t), randn(B, KV, 333, 128).to(t)
    run_attn(ops, "attn many rows: head-major cache", q, kc.transpose(1, 2), vc.transpose(1, 2), 5, k_len=ints(*[333 - 16 * b for b in range(B)]))


def test_attn_many_rows_large_and_equal_scores(ops):
    """All scores equal, growing along the keys (the maximum follows again and again), one key that takes all."""
    randn = gen(750)
    B, n_q, n_k, H = 64, 200, 500, 1
    many_rows(B, n_q, n_k, H, H)
    q, v = randn(B, n_q, H, 128), randn(B, n_k, H, 128).to(F16)
    for name, k in (("equal", torch.zeros(B, n_k, H, 128, device="cuda")), ("growing", torch.linspace(0, 8, n_k, device="cuda")[None, :, None, None] * torch.sign(q[:, :1])),
                    ("one key", randn(B, n_k, H, 128) * (torch.arange(n_k, device="cuda") == 333)[None, :, None, None] * 12)):
        for t in (F16, BF16):
            run_attn(ops, "attn many rows: scores " + name, q.to(t), k.to(t), v.to(t), 6, norm=False)


# ---------------------------------------------------------------------------------------------------------- linear_act
DT = {F16: DTYPE_F16, BF16: DTYPE_BF16, F8: DTYPE_F8}


def scratch(m, n, k, t, f32, aligned=True):
    return lib.svd_linear_act_ws_bytes(m, n, k, LIN_OUT_F32 if f32 else 0, DT[t], int(aligned))


#        256-row tiles, their last round split; 128-row tiles (all or the last round of them); odd widths that leave element by element; unaligned rows, copied behind the partial sums
SPLIT = [(8448, 2176, 2240), (1100, 1040, 2064), (1100, 1042, 2064), (1101, 1041, 2067), (8449, 2177, 2245)]


@pytest.mark.parametrize("f32", [False, True], ids=["to16", "to32"])
@pytest.mark.parametrize("t", [F16, BF16, F8], ids=str)
@pytest.mark.parametrize("m,n,k", SPLIT)
def test_linear_split_products_with_the_whole_epilogue(ops, m, n, k, t, f32):
    """Scales, bias, activation and residual on tiles whose K is split, compared on rows of every 32-row band of every tile."""
    assert scratch(m, n, k, t, f32) > 0, "K is split"
    randn, x, w, sx, sw = make_linear(800 + k, m, n, k, t)
    e = BF16 if t == F8 else t
    bias, res = randn(n), randn(m, n).to(F32 if f32 else e)
    got = ops.linear_act(x, w, bias=bias, act="gelu_tanh" if f32 else "gelu", residual=res, x_scale=sx, w_scale=sw, out_dtype=F32 if f32 else e)
    part = torch.cat([torch.arange(0, m, 29, device="cuda"), torch.arange(m - 33, m, device="cuda")])
    check_linear(f"linear split {m}x{n}x{k} {t}", got[part], x.float()[part].to(t), w, sx[part] if sx is not None else None, sw, bias, "gelu_tanh" if f32 else "gelu", res[part])
    again = ops.linear_act(x, w, bias=bias, act="gelu_tanh" if f32 else "gelu", residual=res, x_scale=sx, w_scale=sw, out_dtype=F32 if f32 else e)
    assert torch.equal(again, got)
    y = res.clone()
    ops.linear_act(x, w, bias=bias, act="gelu_tanh" if f32 else "gelu", residual=y, x_scale=sx, w_scale=sw, out=y)
    assert torch.equal(y, got), "onto the residual in place"


@pytest.mark.parametrize("f32", [False, True], ids=["to16", "to32"])
@pytest.mark.parametrize("t", [F16, BF16, F8], ids=str)
@pytest.mark.parametrize("m,n,k", SPLIT + [(4100, 2064, 208), (4096, 2048, 320)])
def test_linear_picks_rows_and_columns_in_16_bits(ops, m, n, k, t, f32):
    """One-hot rows select columns of W, small whole numbers that every type holds: any swapped lane, row, column pair or K chunk shows as another number, exactly."""
    x = torch.zeros(m, k, device="cuda")
    idx = (torch.arange(m, device="cuda") * 7) % k
    x[torch.arange(m, device="cuda"), idx] = 1
    w = ((torch.arange(n * k, device="cuda") * 37) % 31 - 15).reshape(n, k).float().to(t)
    res = ((torch.arange(m * n, device="cuda") * 11) % 64 * 4).reshape(m, n).to(F32 if f32 else BF16 if t == F8 else t)
    want = w.float().t()[idx]
    got = ops.linear_act(x.to(t), w, out_dtype=res.dtype)
    assert torch.equal(got.float(), want)
    b = torch.arange(n, device="cuda").remainder(5).float()
    got = ops.linear_act(x.to(t), w, bias=b, act="relu", out_dtype=res.dtype)
    assert torch.equal(got.float(), (want + b).clamp_min(0))
    got = ops.linear_act(x.to(t), w, residual=res, out_dtype=res.dtype)
    assert torch.equal(got.float(), (want + res.float()).to(res.dtype).float())


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu", "relu"])
@pytest.mark.parametrize("m,n,k", [(300, 160, 320), (1100, 1040, 2064), (1100, 1041, 2064)])
def test_linear_tiles_rows_do_not_mix(ops, act, m, n, k):
    """A row of NaN stays in its row, a weight row of NaN in its column, under every activation and in the join too."""
    randn, x, w, _, _ = make_linear(850, m, n, k, BF16)
    clean = ops.linear_act(x, w, act=act)
    x[2], w[7] = float("nan"), float("nan")
    got = ops.linear_act(x, w, act=act)
    nan = torch.isnan(got)
    assert nan[2].all() and nan[:, 7].all() and nan.sum().item() == m + n - 1
    assert torch.equal(got[~nan], clean[~nan])


def test_linear_split_on_two_streams_and_in_graphs(ops):
    """Products with scratch memory (a split K, copies of unaligned rows) on two streams at once, and in two graphs replayed in turn with eager calls in between: bit for bit."""
    cases = []
    for i, (m, n, k, t) in enumerate([(1100, 1040, 2064, BF16), (1101, 1041, 2067, F8)]):
        randn, x, w, sx, sw = make_linear(860 + i, m, n, k, t)
        cases.append((x, w, sx, sw, ops.linear_act(x, w, x_scale=sx, w_scale=sw, act="silu", out_dtype=BF16)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                x, w, sx, sw, _ = cases[s]
                got[s].append(ops.linear_act(x, w, x_scale=sx, w_scale=sw, act="silu", out_dtype=BF16))
    torch.cuda.synchronize()
    for s in range(2):
        assert all(torch.equal(g, cases[s][4]) for g in got[s])
    graphs = []
    for x, w, sx, sw, _ in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.linear_act(x, w, x_scale=sx, w_scale=sw, act="silu", out_dtype=BF16)
        graphs.append((g, y))
    for rep in range(4):
        for (x, w, sx, sw, _), (g, y) in zip(cases, graphs):
            x.copy_(gen(870 + rep)(*x.shape).to(x.dtype))
            eager = ops.linear_act(x, w, x_scale=sx, w_scale=sw, act="silu", out_dtype=BF16).clone()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)
