"""A step's logits to its tokens on the GPU: penalties, biases and masks bit for bit against float32
step by step, sampled tokens against the definition in 64 bits, and the whole run from hidden rows
through a 4-bit LM head, eager and captured."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import q4_helpers as ref

pytestmark = pytest.mark.gpu


def up(dev, a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def rules_of(ie, dev, r):
    put = lambda v: None if v is None else tuple(up(dev, a) for a in v) if isinstance(v, tuple) else up(dev, v)
    r = dict(r)
    if r.get("mask") is not None:
        r["mask"] = r["mask"].view(np.int32)
    return ie.logit_rules(**{k: put(v) for k, v in r.items()})


def draw_rules(rng, R, n, history=200, biases=30, masked=True):
    f32 = lambda a: a.astype(np.float32)
    length = rng.integers(0, history + 1, R).astype(np.int32)
    blen = rng.integers(0, biases + 1, R).astype(np.int32)
    return dict(
        history=((rng.random(R * history) ** 3 * n).astype(np.int32),
                 (np.arange(R) * history).astype(np.int32), length),
        prompt_len=rng.integers(-1, history, R).astype(np.int32),
        repetition=f32(1 + rng.random(R)), presence=f32(rng.random(R)), frequency=f32(rng.random(R)),
        bias=(rng.integers(0, n, R * biases).astype(np.int32), f32(rng.standard_normal(R * biases) * 9),
              (np.arange(R) * biases).astype(np.int32), blen),
        mask=rng.integers(0, 2 ** 32, (max(R // 2, 1), -(-n // 32)), dtype=np.uint32) if masked else None,
        mask_row=rng.integers(-2, R, R).astype(np.int32) if masked else None)


def check(ie, dev, logits, rules, in_place):
    l = up(dev, logits)
    out = l if in_place else torch.full_like(l, float("nan"))
    ie.adjust_logits(out, l, rules_of(ie, dev, rules))
    got = out.cpu().numpy()
    want = ref.adjust(logits, rules)
    assert np.array_equal(got, want, equal_nan=True)
    finite = np.isfinite(want)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    # Four steps rounded to 2^-24 of the largest number met on the way, against 64 bits.
    exact = ref.adjust(logits, rules, np.float64)
    far = np.abs(got[finite] - exact[finite])
    assert (far <= 2.0 ** -20 * (np.abs(logits[finite]) + np.abs(exact[finite]) + 64)).all()
    return l, out


@pytest.mark.parametrize("R,n", [(1, 1), (1, 31), (2, 33), (3, 1000), (1, 8192), (2, 8193), (5, 16385),
                                 (64, 5001), (3, 151936), (1, 262147)])
@pytest.mark.parametrize("in_place", [False, True])
def test_adjust(ie, dev, R, n, in_place):
    print(f"adjust_logits {R} x {n}", flush=True)
    rng = np.random.default_rng(R + n)
    logits = (rng.standard_normal((R, n)) * 6).astype(np.float32)
    check(ie, dev, logits, draw_rules(rng, R, n), in_place)


@pytest.mark.parametrize("only", ["history", "bias", "mask", "none"])
def test_adjust_one_rule(ie, dev, only):
    rng = np.random.default_rng(1)
    R, n = 6, 10007
    every = draw_rules(rng, R, n, 3000, 300)
    names = {"history": ("history", "repetition"), "bias": ("bias",), "mask": ("mask", "mask_row"),
             "none": ()}[only]
    logits = (rng.standard_normal((R, n)) * 6).astype(np.float32)
    check(ie, dev, logits, {k: every[k] for k in names}, False)


def test_adjust_odd_entries(ie, dev):
    """Ids and ranges outside what is there are skipped, values that are not numbers kept as the
    formula leaves them, the later of two biases stands, masks win."""
    n, R = 300, 3
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((R, n)).astype(np.float32)
    logits[0, :6] = [np.inf, -np.inf, np.nan, 0.0, -0.0, 5.0]
    hist = np.array([0, 1, 2, 3, 4, 5, -1, n, 2 ** 31 - 1, -2 ** 31, 5, 5], np.int32)
    rules = dict(history=(hist, np.array([0, -4, 10], np.int32), np.array([12, 8, 2 ** 31 - 1], np.int32)),
                 repetition=np.array([2, 1.5, 1.25], np.float32),
                 frequency=np.array([0.5, 0.25, 0.1], np.float32),
                 presence=np.array([0.3, -0.2, 0.7], np.float32),
                 bias=(np.array([7, 7, 9, -5, n, 7], np.int32), np.array([1, 2, -100, 4, 5, 3], np.float32),
                       np.array([0, 3, -2], np.int32), np.array([3, 100, 5], np.int32)),
                 mask=np.array([[0xFFFFFFFF] * 10, [0] * 10], np.uint32),
                 mask_row=np.array([0, 5, 1], np.int32))
    # 2^31 - 1 entries of a history of 12: only those that are there are read.
    small = dict(rules, history=(hist, rules["history"][1], np.array([12, 8, 2], np.int32)))
    l = up(dev, logits)
    out = torch.full_like(l, float("nan"))
    ie.adjust_logits(out, l, rules_of(ie, dev, rules))
    want = ref.adjust(logits, small)
    assert np.array_equal(out.cpu().numpy(), want, equal_nan=True)
    assert np.isneginf(want[2]).all()


def test_adjust_leaves_other_rows(ie, dev):
    """Rows behind the last one stay as they were."""
    rng = np.random.default_rng(4)
    n = 9000
    logits = rng.standard_normal((5, n)).astype(np.float32)
    l, out = up(dev, logits), torch.full((5, n), 7.0, device=dev)
    rules = draw_rules(rng, 3, n)
    ie.adjust_logits(out[:3], l[:3], rules_of(ie, dev, rules))
    got = out.cpu().numpy()
    assert np.array_equal(got[:3], ref.adjust(logits[:3], rules)) and (got[3:] == 7).all()


# ------------------------------------------------------------------ sampling ----
def rows_of_logits(rng, R, n):
    l = (rng.standard_normal((R, n)) * 2.5).astype(np.float32)
    for r in range(R):
        at = rng.integers(0, n, 12)
        l[r, at] = rng.random(12) * 12 + 2
    return l


def draw(ie, dev, l, t, u, k=None, p=None, m=None, ws=None):
    R, n = l.shape
    put = lambda a, d: None if a is None else up(dev, np.asarray(a, d))
    out = torch.full((R,), -7, dtype=torch.int32, device=dev)
    ie.sample_rows(out, up(dev, l), put(t, np.float32), put(u, np.float32), put(k, np.int32),
                   put(p, np.float32), put(m, np.float32),
                   workspace=ie.sample_rows_workspace(R, n, dev) if ws is None else ws)
    return out.cpu().numpy()


def expect(l, t, u, k=None, p=None, m=None):
    get = lambda a, r, d: d if a is None else a[r]
    return [ref.sample(l[r], t[r], u[r], get(k, r, 0), get(p, r, 1.0), get(m, r, 0.0))
            for r in range(l.shape[0])]


SIZES = [(1, 1), (2, 2), (3, 63), (4, 64), (7, 65), (33, 1000), (64, 4099), (9, 32000), (1, 151936),
         (16, 151936), (2, 300001)]


@pytest.mark.parametrize("R,n", SIZES)
@pytest.mark.parametrize("mode", ["plain", "k", "p", "m", "all"])
def test_sample(ie, dev, R, n, mode):
    print(f"sample_rows {R} x {n}, {mode}", flush=True)
    rng = np.random.default_rng(R + n)
    l = rows_of_logits(rng, R, n)
    t, u = 0.3 + 1.5 * rng.random(R), rng.random(R)
    k = np.exp(rng.random(R) * np.log(n + 1)).astype(np.int32) if mode in ("k", "all") else None
    p = rng.random(R) if mode in ("p", "all") else None
    m = rng.random(R) ** 3 if mode in ("m", "all") else None
    assert draw(ie, dev, l, t, u, k, p, m).tolist() == expect(l, t, u, k, p, m)


@pytest.mark.parametrize("n", [5, 1000, 20011, 151936])
def test_sample_ties(ie, dev, n):
    """Equal logits: a prefix by index of exactly the right length; two levels; zeros of both signs."""
    rng = np.random.default_rng(n)
    l = np.zeros((8, n), np.float32)
    l[1::2] = (rng.random((4, n)) < 0.3).astype(np.float32)
    l[4, ::2] = -0.0
    t, u = np.ones(8), np.array([0.0, 0.3, 0.5, 0.7, 0.999, 1 - 2.0 ** -24, 0.1, 0.9])
    for p in (0.25, 0.5, 0.9, 1e-9):
        assert draw(ie, dev, l, t, u, p=[p] * 8).tolist() == expect(l, t, u, p=[p] * 8)
    for k in (1, 2, n // 2, n - 1, n):
        kk = [k] * 8
        assert draw(ie, dev, l, t, u, k=kk).tolist() == expect(l, t, u, k=kk)
        assert draw(ie, dev, l, t, u, k=kk, p=[0.5] * 8).tolist() == expect(l, t, u, k=kk, p=[0.5] * 8)


@pytest.mark.parametrize("many", [6143, 6144, 6145, 32767, 32768, 32769])
def test_sample_border_of_many_tokens(ie, dev, many):
    """So many tokens of two near logits at random places, all in one bin, the others far below: what
    a border's list holds in LDS, in the workspace, and not at all."""
    n = 40007
    rng = np.random.default_rng(many)
    l = np.full((6, n), -50, np.float32)
    for r in range(6):
        at = rng.permutation(n)[:many]
        l[r, at] = np.where(rng.random(many) < 0.5, 1.0, np.float32(1.0 + 2.0 ** -20))
    t, u = np.ones(6), rng.random(6)
    k = np.array([1, 2, many // 3, many - 1, many, many + 1], np.int32)
    p = np.array([1e-6, 0.2, 0.5, 0.75, 0.999, 0.4])
    m = np.full(6, 0.1)
    assert draw(ie, dev, l, t, u, k=k).tolist() == expect(l, t, u, k=k)
    assert draw(ie, dev, l, t, u, p=p).tolist() == expect(l, t, u, p=p)
    assert draw(ie, dev, l, t, u, k, p, m).tolist() == expect(l, t, u, k, p, m)


@pytest.mark.parametrize("n", [7, 5000, 151936])
def test_sample_odd_values(ie, dev, n):
    """Settings and random numbers outside their ranges; rows of nothing, of one token, of
    infinities, with NaN; temperatures from tiny to infinite."""
    rng = np.random.default_rng(n)
    l = np.repeat(rows_of_logits(rng, 1, n), 16, 0)
    l[1] = -np.inf
    l[2] = np.nan
    l[3] = -np.inf
    l[3, n // 2] = 1.0
    l[4, [1, n - 1]] = np.inf
    l[5, ::2] = np.nan
    l[6, 3:] = -np.inf
    l[7] = 3.0e38
    l[8] *= -1e37 / np.abs(l[8]).max()
    t = np.array([0, 1, 1, 1, 1, 1, 1, 1, 1e36, 1e-40, np.inf, np.nan, -1, 1, 1, 1], np.float32)
    u = np.array([.5, .5, .5, .5, .75, .5, .4, .6, .5, .5, .3, .5, .5, 1.0, -1, np.nan], np.float32)
    want = expect(l, t, u)
    assert want[1] == want[2] == 0 and want[4] == n - 1
    assert draw(ie, dev, l, t, u).tolist() == want
    k = np.array([0, 5, 5, 5, 1, 3, 2, 4, 0, -1, 2 ** 31 - 1, 1, 1, 1, 2, 3], np.int32)
    p = np.array([.5, .5, .5, .5, .5, .9, .5, .3, -1, 0, .2, np.nan, 2, np.inf, -np.inf, .7], np.float32)
    m = np.array([.5, .5, .5, .5, .5, .1, 1, 0, -1, 2, 1, np.nan, 2, np.inf, -np.inf, .7], np.float32)
    m0 = np.where(np.isnan(m), 0, m)
    p0 = np.where(np.isnan(p), 1, p)
    assert draw(ie, dev, l, t, u, k, p, m).tolist() == expect(l, t, u, k, p0, m0)


def test_sample_greedy_is_argmax(ie, dev):
    rng = np.random.default_rng(8)
    l = np.round(rows_of_logits(rng, 20, 3001))  # ties
    out = torch.empty((20,), dtype=torch.int32, device=dev)
    ie.argmax_rows(out, up(dev, l))
    got = draw(ie, dev, l, np.zeros(20), rng.random(20))
    assert got.tolist() == out.cpu().tolist()
    assert draw(ie, dev, l, np.ones(20), rng.random(20), k=np.ones(20)).tolist() == got.tolist()


def test_sample_does_not_depend_on_the_batch(ie, dev):
    rng = np.random.default_rng(6)
    R, n = 40, 30011
    l, t, u = rows_of_logits(rng, R, n), 0.5 + rng.random(R), rng.random(R)
    k, p, m = rng.integers(0, 200, R), 0.5 + rng.random(R) * 0.6, rng.random(R) * 0.05
    every = draw(ie, dev, l, t, u, k, p, m)
    for a, b in ((0, 1), (5, 6), (3, 20), (39, 40)):
        s = slice(a, b)
        assert draw(ie, dev, l[s], t[s], u[s], k[s], p[s], m[s]).tolist() == every[s].tolist()


def test_sample_frequencies(ie, dev):
    """An even sweep of u gives each token its probability to one part of the sweep."""
    l = np.log(np.array([1, 2, 3, 4, 6], np.float32))
    R = 1600
    got = draw(ie, dev, np.repeat(l[None], R, 0), np.ones(R), (np.arange(R) + 0.5) / R)
    assert np.abs(np.bincount(got, minlength=5) - np.array([1, 2, 3, 4, 6]) * R / 16).max() <= 1


# -------------------------------------------------- hidden rows to tokens ----
class Run:
    """Decode steps from hidden rows: final norm, 4-bit LM head, rules, token; the token joins its
    row's history on the device, as an engine keeps it."""

    def __init__(self, ie, dev, R, n, cols, room, seed):
        rng = self.rng = np.random.default_rng(seed)
        self.ie, self.dev, self.R, self.n, self.cols = ie, dev, R, n, cols
        packed, s, z, self.w = ref.quantize(rng, n, cols, 64, "f16", True)
        self.head = ie.matrix_q4(up(dev, packed), up(dev, s), 64, zero=up(dev, z))
        self.norm = torch.ones(cols, device=dev)
        self.prompt = rng.integers(1, 6, R).astype(np.int32)
        self.hist0 = rng.integers(0, n, (R, room)).astype(np.int32)
        f32 = lambda a: a.astype(np.float32)
        self.plain = dict(
            prompt_len=self.prompt, repetition=f32(1 + rng.random(R) * .4), presence=f32(rng.random(R)),
            frequency=f32(rng.random(R)),
            bias=(rng.integers(0, n, 2 * R).astype(np.int32), f32(rng.standard_normal(2 * R) * 3),
                  (2 * np.arange(R)).astype(np.int32), np.full(R, 2, np.int32)),
            mask=rng.integers(0, 2 ** 32, (R, -(-n // 32)), dtype=np.uint32),
            mask_row=np.where(rng.random(R) < .5, np.arange(R), -1).astype(np.int32))
        self.hist, self.len = up(dev, self.hist0), up(dev, self.prompt)
        self.start = (np.arange(R) * room).astype(np.int32)
        t = lambda k: up(dev, self.plain[k])
        self.rules = ie.logit_rules(
            history=(self.hist, up(dev, self.start), self.len), prompt_len=t("prompt_len"),
            repetition=t("repetition"), presence=t("presence"), frequency=t("frequency"),
            bias=tuple(up(dev, a) for a in self.plain["bias"]),
            mask=up(dev, self.plain["mask"].view(np.int32)), mask_row=t("mask_row"))
        self.t, self.k = f32(.5 + rng.random(R)), rng.integers(0, 60, R).astype(np.int32)
        self.p, self.m = f32(.7 + .4 * rng.random(R)), f32(.05 * rng.random(R))
        self.dt, self.dk, self.dp, self.dm = (up(dev, a) for a in (self.t, self.k, self.p, self.m))
        self.x, self.u = torch.zeros((R, cols), device=dev), torch.zeros(R, device=dev)
        self.xn = torch.empty_like(self.x)
        self.raw, self.logits = torch.empty((R, n), device=dev), torch.empty((R, n), device=dev)
        self.tokens = torch.empty(R, dtype=torch.int32, device=dev)
        self.ws = ie.matmul_q4_workspace(R, cols, dev), ie.sample_rows_workspace(R, n, dev)

    def step(self):
        ie = self.ie
        ie.rmsnorm(self.xn, self.x, self.norm, 1e-6)
        ie.matmul_q4(self.raw, self.xn, self.head, workspace=self.ws[0])
        ie.adjust_logits(self.logits, self.raw, self.rules)
        ie.sample_rows(self.tokens, self.logits, self.dt, self.u, self.dk, self.dp, self.dm,
                       workspace=self.ws[1])
        self.hist.scatter_(1, self.len.long()[:, None], self.tokens[:, None])
        self.len += 1

    def feed(self):
        self.x.copy_(up(self.dev, self.rng.standard_normal((self.R, self.cols), dtype=np.float32)))
        self.u.copy_(up(self.dev, self.rng.random(self.R).astype(np.float32)))

    def check(self, hist, length):
        """One step done on host copies of the history before it."""
        x = self.x.cpu().numpy().astype(np.float64)
        xn = x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-6)
        raw = self.raw.cpu().numpy()
        tol = ref.sum_tolerance(self.cols, 64, self.w, xn) * 1.1 + 2.0 ** -20 * np.abs(xn @ self.w.T)
        assert (np.abs(raw - xn @ self.w.T) <= tol + 1e-6).all()
        rules = dict(self.plain, history=(hist, self.start, length))
        logits = self.logits.cpu().numpy()
        assert np.array_equal(logits, ref.adjust(raw, rules))
        want = expect(logits, self.t, self.u.cpu().numpy(), self.k, self.p, self.m)
        assert self.tokens.cpu().tolist() == want
        hist = hist.copy()
        hist[np.arange(self.R), length] = want
        assert np.array_equal(self.hist.cpu().numpy(), hist)
        return hist, length + 1


@pytest.mark.parametrize("R,n,cols", [(1, 5000, 256), (7, 3001, 896), (24, 20000, 128)])
def test_hidden_rows_to_tokens(ie, dev, R, n, cols):
    run = Run(ie, dev, R, n, cols, 20, R)
    hist, length = run.hist0, run.prompt
    for _ in range(4):
        run.feed()
        run.step()
        hist, length = run.check(hist, length)


def test_two_captured_runs_in_turn(ie, dev):
    """Two runs recorded into graphs of their own, replayed in turn with eager work between."""
    runs = [Run(ie, dev, 5, 9000, 256, 24, 11), Run(ie, dev, 20, 2100, 512, 24, 12)]
    state, graphs = [], []
    for r in runs:
        r.feed()
        r.step()  # warms up, eagerly
        state.append(r.check(r.hist0, r.prompt))
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            r.step()
        graphs.append(g)
    for _ in range(4):
        for i, (r, g) in enumerate(zip(runs, graphs)):
            r.feed()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            state[i] = r.check(*state[i])
            torch.randn(1000, device=dev).sum().item()


@pytest.mark.parametrize("t", [0.02, 0.1, 0.3, 1.0, 4.0, 60.0])
def test_sample_cold_hot_and_masked(ie, dev, t):
    """Rows whose borders lie where weights vanish (cold), in one wide bin (hot), or past all that a
    grammar leaves."""
    rng = np.random.default_rng(int(t * 100))
    R, n = 12, 60001
    l = rows_of_logits(rng, R, n)
    for r in range(0, R, 3):
        l[r, rng.random(n) < 0.9995] = -np.inf
    l[1] = -np.inf
    l[1, 77] = -3
    tt, u = np.full(R, t, np.float32), rng.random(R)
    k = rng.integers(1, 400, R)
    p, m = 0.5 + 0.5 * rng.random(R), 10.0 ** -rng.integers(1, 16, R)
    for kk, pp, mm in ((k, None, None), (None, p, None), (None, None, m), (k, p, None), (k, None, m),
                       (None, p, m), (k, p, m), (k * 100, p, m)):
        assert draw(ie, dev, l, tt, u, kk, pp, mm).tolist() == expect(l, tt, u, kk, pp, mm)


def test_sample_wide_borders(ie, dev):
    """min-p and top-k borders in the thick of a row, among more tokens than a few bins are listed for,
    alone and under top-p."""
    rng = np.random.default_rng(77)
    R, n = 8, 151936
    l = (rng.standard_normal((R, n)) * 2.5).astype(np.float32)
    l[::2] = np.round(l[::2] * 4) / 4  # few values, thousands of tokens each
    t, u = np.full(R, 1.5, np.float32), rng.random(R)
    m, p, k = 10.0 ** -rng.uniform(1, 5, R), 0.3 + 0.69 * rng.random(R), rng.integers(2000, 140000, R)
    for kk, pp, mm in ((None, None, m), (None, p, m), (k, None, None), (k, p, None), (k, p, m), (None, p, None)):
        assert draw(ie, dev, l, t, u, kk, pp, mm).tolist() == expect(l, t, u, kk, pp, mm)


def test_sample_largest_vocabulary(ie, dev):
    """4,194,304 tokens, a row of few values and one of many; one more token is refused."""
    rng = np.random.default_rng(4)
    n = 1 << 22
    l = np.zeros((2, n), np.float32)
    l[0, rng.integers(0, n, n // 3)] = 1.0
    l[1] = rng.standard_normal(n, dtype=np.float32)
    t, u = np.ones(2), np.array([0.83, 0.41])
    for k, p in ((None, None), ([1500000, 0], [1.0, 0.4]), ([3000000, 7], [0.6, 0.9])):
        assert draw(ie, dev, l, t, u, k, p).tolist() == expect(l, t, u, k, p)
    assert ie.lib().ie_hip_sample_rows_workspace_bytes(1, n + 1) == 0
    big = torch.zeros((1, n + 1), device=dev)
    one = torch.zeros(1, device=dev)
    with pytest.raises(ie.IeHipError, match="4,194,304"):
        ie.sample_rows(torch.zeros(1, dtype=torch.int32, device=dev), big, one, one,
                       workspace=ie.sample_rows_workspace(1, n, dev))


def test_two_streams_at_once(ie, dev):
    """Calls on two streams with workspaces of their own, and a workspace made for more rows."""
    rng = np.random.default_rng(21)
    R, n = 16, 70001
    ls = [rows_of_logits(rng, R, n) for _ in range(2)]
    t, u, p = 0.5 + rng.random(R), rng.random(R), 0.5 + 0.5 * rng.random(R)
    f32 = lambda a: up(dev, np.asarray(a, np.float32))
    dl, dt, du, dp = [up(dev, l) for l in ls], f32(t), f32(u), f32(p)
    ws = [ie.sample_rows_workspace(64, 100000, dev) for _ in range(2)]
    outs = [torch.full((R,), -1, dtype=torch.int32, device=dev) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i in range(2):
            ie.sample_rows(outs[i], dl[i], dt, du, top_p=dp, workspace=ws[i], stream=streams[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert outs[i].tolist() == expect(ls[i], t, u, None, p)


def test_calls_refuse_what_does_not_fit(ie, dev):
    z = lambda *s, **k: torch.zeros(*s, device=dev, **k)
    i32 = torch.int32
    l, one = z(2, 100), z(2)
    out = z(2, dtype=i32)
    for bad in (dict(workspace=None), dict(workspace=z(16, dtype=torch.uint8)), dict(top_k=z(3, dtype=i32)),
                dict(top_p=z(2, dtype=torch.float64)), dict(min_p=z(2, 1))):
        with pytest.raises(ie.IeHipError):
            ie.sample_rows(out, l, one, one, **{"workspace": ie.sample_rows_workspace(2, 100, dev), **bad})
    with pytest.raises(ie.IeHipError, match="contiguous"):
        ie.sample_rows(out, z(100, 2).t(), one, one, workspace=ie.sample_rows_workspace(2, 100, dev))
    with pytest.raises(ie.IeHipError, match="words"):
        ie.adjust_logits(l, l, ie.logit_rules(mask=z(2, 3, dtype=i32)))
    rules = ie.logit_rules(history=(z(4, dtype=i32), z(3, dtype=i32), z(3, dtype=i32)))
    with pytest.raises(ie.IeHipError, match="rows"):
        ie.adjust_logits(l, l, rules)
    with pytest.raises(ie.IeHipError, match="shape"):
        ie.adjust_logits(z(2, 99), l, ie.logit_rules())
    w = ie.matrix_q4(z(16, 16, dtype=torch.uint8), z(16, 1), 32)
    x, y = z(40, 32), z(40, 16)
    with pytest.raises(ie.IeHipError, match="workspace"):
        ie.matmul_q4(y, x, w)
    for args in ((z(40, 15), x, w), (y, z(40, 64), w), (z(39, 16), x, w), (y, x, w, z(15)),
                 (y, x.cpu(), w), (y.cpu(), x, w), (y.half(), x, w)):
        with pytest.raises(ie.IeHipError):
            ie.matmul_q4(*args, workspace=ie.matmul_q4_workspace(40, 32, dev))
    ie.matmul_q4(z(0, 16), z(0, 32), w)
    ie.sample_rows(z(0, dtype=i32), z(0, 100), z(0), z(0))
    vec = z(16) + 9
    ie.matmul_q4(vec, z(32), w)  # one token as a vector
    assert not vec.any()
