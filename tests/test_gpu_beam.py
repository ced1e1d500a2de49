"""gkv_beam_select on the GPU: tokens and parents exactly, scores to their last fp32 bit or the sums'
error, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
NEG = -np.inf


def plain(x):
    """What a logit counts as."""
    x = np.asarray(x, np.float64)
    big = float(np.finfo(np.float32).max)
    return np.where(np.isnan(x), NEG, np.minimum(x, big))


def expect(x, cum, K, n, done=None, eos=-1):
    """Scores (64 bits), parents, tokens, done."""
    rows, V = x.shape
    x, cum = plain(x), plain(cum)
    z = np.full((rows, V), NEG)
    for r in range(rows):
        if done is not None and done[r]:
            z[r, eos] = cum[r]
            continue
        m = x[r].max()
        if cum[r] > NEG and m > NEG:
            # (a row's n largest logits compete: next to a cum beyond 2^53 of their differences,
            # which no sum of log-probabilities is, scores of unequal logits are equal in 64 bits)
            top = np.lexsort((np.arange(V), -x[r]))[:n]
            z[r, top] = cum[r] + (x[r, top] - (m + np.log(np.exp(x[r] - m).sum())))
    out = []
    for q in range(rows // K):
        flat = z[q * K:q * K + K].reshape(-1)
        at = np.lexsort((np.arange(flat.size), -flat))[:n]
        row, t = q * K + at // V, at % V
        d = (t == eos) | (np.zeros(n, bool) if done is None else np.asarray(done)[row] != 0)
        out.append((flat[at], row, t, d))
    return [np.stack([o[i] for o in out]) for i in range(4)]


def run(gkv, x, cum, K, n, done=None, eos=-1, stream=None, ws=None):
    """x: a device tensor [rows, V]."""
    rows, V = x.shape
    R = rows // K
    dev = lambda a, t: torch.from_numpy(np.ascontiguousarray(a, t)).cuda()  # noqa: E731
    i32 = lambda: torch.full((R, n), 77, dtype=torch.int32, device="cuda")  # noqa: E731
    scores, parents, tokens, ended = torch.full((R, n), 7.0, device="cuda"), i32(), i32(), i32()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    if ws is None:
        ws = torch.full((gkv.beam_workspace_bytes(R, K, V, n),), 0xFF, dtype=torch.uint8, device="cuda")
    gkv.beam_select(x, dev(cum, np.float32), K, scores, parents, tokens, done=None if done is None else dev(done, np.int32),
                    eos=eos, done_out=ended, workspace=ws, dev_err=err, stream=stream)
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in (scores, parents, tokens, ended)] + [int(err.item())]


def compare(got, want, V):
    """Scores: the row's sum is off by at most its terms' roundings (2^-24 each in the difference, the
    factor and the exponential, which moves by |d| log2 e of it, |d| < 128: 2^-16; sums of at most 2^11
    terms a lane 2^-13: together under 2^-12), the output by half a step."""
    scores, parents, tokens, ended, err = got
    s, p, t, d = want
    assert np.array_equal(parents, p) and np.array_equal(tokens, t) and np.array_equal(ended, d)
    fin = np.isfinite(s)
    with np.errstate(over="ignore"):
        assert np.array_equal(scores[~fin], s[~fin].astype(np.float32))
    assert (np.abs(scores[fin] - s[fin]) <= 2.0 ** -12 + np.abs(s[fin]) * 2.0 ** -24).all()


def check(gkv, x, cum, K, n, done=None, eos=-1, err=0, dtype=torch.float32):
    t = torch.from_numpy(np.asarray(x, np.float32)).to(dtype).cuda()
    got = run(gkv, t, cum, K, n, done, eos)
    compare(got, expect(t.float().cpu().numpy(), cum, K, n, done, eos), t.shape[1])
    assert got[4] == err


def logits(rng, rows, V, scale=2.5):
    return (rng.standard_normal((rows, V)) * scale).astype(np.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,K,V,n", [(1, 1, 1, 1), (1, 1, 7, 3), (2, 3, 64, 6), (1, 4, 1000, 4), (3, 2, 1025, 64),
                                     (1, 1, 4097, 1), (5, 8, 5003, 16), (1, 64, 300, 64), (2, 2, 40001, 5),
                                     (40, 5, 2048, 10), (1, 2, 150000, 33)])
def test_sizes(gkv, cuda, dtype, R, K, V, n):
    rng = np.random.default_rng(V + n)
    check(gkv, logits(rng, R * K, V), rng.standard_normal(R * K) * 3 - 10, K, n, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits(gkv, cuda, dtype):
    rng = np.random.default_rng(0)
    x = rng.integers(-2, 3, (6, 5000)).astype(np.float32)
    check(gkv, x, np.zeros(6), 3, 40, dtype=dtype)
    check(gkv, np.zeros((4, 3000), np.float32), [-1, -1, -1, -1], 4, 64, dtype=dtype)
    same = np.repeat(logits(rng, 1, 2000), 4, 0)
    check(gkv, same, [-3, -3, -3, -3], 4, 9, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_forbidden_tokens(gkv, cuda, dtype):
    """Rows of which few tokens are left, fewer than asked for, none."""
    rng = np.random.default_rng(1)
    x = np.full((8, 6001), NEG, np.float32)
    low = np.float32(torch.finfo(dtype).min)
    for r, k in enumerate((1, 3, 20, 0)):
        x[r, rng.permutation(6001)[:k]] = logits(rng, 1, k)[0] if k else 0
    x[4:] = low  # masked by the type's lowest value
    for r in (4, 5, 6):
        x[r, rng.permutation(6001)[:r]] = logits(rng, 1, r)[0]
    cum = np.array([-3.0, -5, -1, -2, -4, -1, -2, -7])
    check(gkv, x, cum, 4, 12, dtype=dtype)
    check(gkv, x, cum, 1, 5, dtype=dtype)
    check(gkv, x[3:4], cum[3:4], 1, 5, dtype=dtype)  # a row of -inf alone


def test_lowest_values_alone(gkv, cuda):
    check(gkv, np.full((2, 3000), np.finfo(np.float32).min), [-1, -2], 2, 7)


def test_large_logits(gkv, cuda):
    rng = np.random.default_rng(2)
    x = logits(rng, 4, 3001, 1e30)
    check(gkv, x, [0, 0, 0, 0], 2, 3)
    x = logits(rng, 4, 3001, 100.0)
    check(gkv, x, [0, -50, 3, 1e10], 2, 30)


def test_ended_beams(gkv, cuda):
    rng = np.random.default_rng(3)
    x = logits(rng, 12, 3000)
    x[:, 5] = 9
    done = np.array([0, 1, 0, 1, 1, 1, 1, 0, 0, 0, 0, 0])
    cum = rng.standard_normal(12) * 2 - 8
    check(gkv, x, cum, 4, 8, done=done, eos=5)
    check(gkv, x, cum, 4, 8, eos=5)
    check(gkv, x, cum, 1, 3, done=done, eos=0)
    check(gkv, x, cum, 1, 4, done=done, eos=2999)
    x[done != 0] = np.nan  # not read
    check(gkv, x, cum, 4, 8, done=done, eos=5)


def test_places_without_a_beam(gkv, cuda):
    """A search's first step: one beam, the others have no score."""
    rng = np.random.default_rng(4)
    x = logits(rng, 8, 2500)
    x[1:4] = np.nan
    check(gkv, x, [-2, NEG, NEG, NEG, -1, -1, NEG, -3], 4, 6)
    check(gkv, x[:4], [NEG] * 4, 4, 6)
    check(gkv, x[1:2, :3], [NEG], 1, 3)


def test_nan_and_infinite_logits(gkv, cuda):
    rng = np.random.default_rng(5)
    x = logits(rng, 4, 4100)
    x[0, [0, 7, 4099]] = np.nan
    check(gkv, x, [-1] * 4, 2, 5, err=8)
    x = logits(rng, 2, 4100)
    x[1, 100] = np.inf
    check(gkv, x, [-1] * 2, 2, 5, err=8)
    check(gkv, np.full((2, 900), np.nan, np.float32), [-1, -2], 2, 5, err=8)
    x = logits(rng, 3, 900)
    check(gkv, x, [np.nan, -1, -4], 3, 5, err=8)
    check(gkv, x, [-3, np.inf, -4], 3, 1, err=8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,pad,shift", [(1000, 0, 1), (1001, 3, 0), (4096, 5, 3), (77, 1, 2), (9, 0, 7), (3, 0, 1)])
def test_rows_at_any_alignment(gkv, cuda, dtype, V, pad, shift):
    """Rows inside a larger array, whose neighbours would win."""
    rng = np.random.default_rng(V)
    rows, stride = 6, V + pad
    whole = torch.full((rows * stride + 64,), 1e4, dtype=dtype, device="cuda")
    x = whole[shift:shift + rows * stride].view(rows, stride)[:, :V]
    x.copy_(torch.from_numpy(logits(rng, rows, V)))
    cum = rng.standard_normal(rows)
    got = run(gkv, x, cum, 3, min(V, 8))
    compare(got, expect(x.float().cpu().numpy(), cum, 3, min(V, 8)), V)
    assert got[4] == 0


def test_a_request_alone_gives_the_same(gkv, cuda):
    """However rows are cut among workgroups, the choice is the same."""
    rng = np.random.default_rng(6)
    x = torch.from_numpy(logits(rng, 600, 8000)).cuda()
    cum = rng.standard_normal(600) - 5
    many = run(gkv, x, cum, 6, 12)
    for r in (0, 57, 99):
        one = run(gkv, x[6 * r:6 * r + 6], cum[6 * r:6 * r + 6], 6, 12)
        assert np.array_equal(one[1][0] + 6 * r, many[1][r]) and np.array_equal(one[2][0], many[2][r])
        assert np.abs(one[0][0] - many[0][r]).max() <= 2.0 ** -12


def test_increasing_logits(gkv, cuda):
    """Every logit beats all before it."""
    x = np.arange(20000, dtype=np.float32)[None] * 1e-3
    check(gkv, np.repeat(x, 2, 0), [-1, -1.5], 2, 64)
    check(gkv, np.repeat(-x, 2, 0), [-1, -1.5], 2, 64)


def test_captured_selections_share_a_workspace(gkv, cuda):
    """Two captured calls of one workspace, replayed in turn with other logits."""
    rng = np.random.default_rng(7)
    K, V, n = 4, 5000, 8
    x = [torch.empty(2 * K, V, device="cuda"), torch.empty(3 * K, V, dtype=torch.bfloat16, device="cuda")]
    cum = [torch.zeros(t.shape[0], device="cuda") for t in x]
    out = [[torch.zeros(t.shape[0] // K, n, dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32)]
           for t in x]
    ws = torch.empty(gkv.beam_workspace_bytes(3, K, V, n), dtype=torch.uint8, device="cuda")
    side, graphs = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    for t, c, o in zip(x, cum, out):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            gkv.beam_select(t, c, K, *o, workspace=ws)
    for _ in range(4):
        for t, c in zip(x, cum):
            t.copy_(torch.from_numpy(logits(rng, *t.shape)))
            c.copy_(torch.from_numpy(rng.standard_normal(c.shape[0]).astype(np.float32)))
        for g in graphs:
            g.replay()
        for t, c, o in zip(x, cum, out):
            s, p, tok, _ = expect(t.float().cpu().numpy(), c.cpu().numpy(), K, n)
            assert np.array_equal(o[1].cpu().numpy(), p) and np.array_equal(o[2].cpu().numpy(), tok)
            assert np.abs(o[0].cpu().numpy() - s).max() <= 2.0 ** -12


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_past_32_bit_offsets(gkv, cuda, dtype):
    V, stride = 4001, 2**31 + 7
    x = torch.empty(stride + V, dtype=dtype, device="cuda").as_strided((2, V), (stride, 1))
    x.copy_(torch.from_numpy(logits(np.random.default_rng(5), 2, V)))
    cum = np.array([-1.5, -1.25], np.float32)
    compare(run(gkv, x, cum, 2, 6), expect(x.float().cpu().numpy(), cum, 2, 6), V)
