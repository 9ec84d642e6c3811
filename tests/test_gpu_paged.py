"""The paged 4-bit KV cache on the device: appended bytes, rotated queries and
read rows equal to the definition bit for bit, attention within a tolerance made
of its roundings, at the sizes, masks and strides where each can go wrong."""
import numpy as np
import pytest

from tests import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _t(a, dtype=None):
    import torch
    x = torch.from_numpy(np.ascontiguousarray(a))
    return (x if dtype is None else x.to(dtype)).to(DEV)


def _dtype(name):
    import torch
    return torch.float32 if name == "f32" else torch.bfloat16


class Setup:
    """Sessions [(kv_len, q_len)] over a host pool with shuffled pages, and the
    device's copies of it."""

    def __init__(self, hip, heads, n_kv, hd, sessions, ps=16, vd=None, dtype="f32", seed=0, spare=2, scale=1.0):
        rng = np.random.default_rng(seed)
        self.rng, self.hip, self.heads, self.dtype = rng, hip, heads, dtype
        self.kv_lens = np.array([a for a, _ in sessions], np.int32)
        self.q_starts = np.concatenate([[0], np.cumsum([b for _, b in sessions])]).astype(np.int32)
        pages = [-(-a // ps) for a, _ in sessions]
        n_pages = sum(pages) + spare
        self.table = np.full((len(sessions), max(pages) + 1), -1, np.int32)
        order = rng.permutation(n_pages)
        at = 0
        for i, n in enumerate(pages):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.pool = R.Pool(n_pages, ps, n_kv, hd, vd)
        self.n = int(self.q_starts[-1])
        self.spread = np.exp(0.4 * rng.standard_normal((n_kv, hd))) * scale

    def round(self, x):
        x = np.asarray(x, np.float32)
        return R.bf16_round(x) if self.dtype == "bf16" else x

    def randn(self, *shape):
        return self.rng.standard_normal(shape).astype(np.float32)

    def fill(self, skip_rows=False):
        """Stores every cached position of every session (without the batch's own
        rows if skip_rows)."""
        p = self.pool
        for s, n in enumerate(self.kv_lens):
            last = n - (self.q_starts[s + 1] - self.q_starts[s]) if skip_rows else n
            for t in range(max(0, last)):
                page = self.table[s, t // p.ps]
                p.store("k", page, t % p.ps, self.randn(p.n_kv, p.hd) * self.spread.astype(np.float32))
                p.store("v", page, t % p.ps, self.randn(p.n_kv, p.vd) * np.float32(0.5))
        return self

    def upload(self, max_q=None, max_kv=None):
        p, hip = self.pool, self.hip
        self.k_dev, self.v_dev = _t(p.k), _t(p.v)
        self.cache = hip.PagedKv(self.k_dev, self.v_dev, p.n_pages, p.ps, p.n_kv, p.hd, p.vd)
        most = max(1, int(np.diff(self.q_starts).max(initial=1)))
        self.t_table, self.t_lens, self.t_starts = _t(self.table), _t(self.kv_lens), _t(self.q_starts)
        self.batch = hip.PagedBatch(self.t_table, self.t_lens, self.t_starts, max_q or most,
                                    int(self.kv_lens.max()) if max_kv is None else max_kv)
        return self

    def workspace(self, n_rows):
        import torch
        n = self.hip.paged_attention_workspace(self.cache, self.batch, n_rows, self.heads)
        # NaN bytes: what a join reads without a split having written it shows
        return torch.full((n,), 0xFF, dtype=torch.uint8, device=DEV) if n else None

    def attend(self, q, window=0, sinks=None, scale=None, rows=None):
        """Checked attention of host queries [rows][heads][hd]; returns the output."""
        import torch
        p = self.pool
        scale = p.hd ** -0.5 if scale is None else scale
        n = q.shape[0]
        out = torch.full((n, self.heads, p.vd), 7.0, dtype=_dtype(self.dtype), device=DEV)
        assert self.hip.paged_attention_dev(self.cache, self.batch, _t(q, _dtype(self.dtype)), out, scale,
                                            self.workspace(n), None if sinks is None else _t(sinks), window)
        got = out.float().cpu().numpy().astype(np.float64)
        ref, spread, size = R.attention(p, self.table, self.kv_lens, self.q_starts, q, np.float32(scale), window,
                                        sinks)
        rows = slice(0, self.n) if rows is None else rows
        tol = R.tolerance(ref, spread, size, self.dtype)
        bad = ~(np.abs(got - ref) <= tol)[rows]
        assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got - ref)[rows].max(), tol[rows].max())
        return got


# ---- attention: head layouts, lengths, masks -----------------------------------------
SHAPES = [  # heads, kv heads, head dim, value dim
    (4, 4, 64, 64), (8, 2, 128, 128), (5, 1, 128, 128), (16, 2, 64, 64), (16, 1, 128, 128), (20, 1, 64, 64),
    (4, 2, 256, 256), (16, 1, 256, 256), (6, 2, 80, 80), (3, 3, 96, 40), (2, 1, 8, 16), (8, 1, 192, 128), (2, 2, 40, 200),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,n_kv,hd,vd", SHAPES)
def test_single_tokens(hip, heads, n_kv, hd, vd, dtype):
    s = Setup(hip, heads, n_kv, hd, [(1, 1), (15, 1), (16, 1), (17, 1), (64, 1), (65, 1), (131, 1)], vd=vd, dtype=dtype,
              seed=heads + hd).fill().upload()
    s.attend(s.round(1.5 * s.randn(s.n, heads, hd)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,n_kv,hd,vd", [(8, 2, 128, 128), (16, 2, 64, 64), (5, 1, 128, 128), (4, 2, 256, 256),
                                              (20, 1, 64, 64), (4, 4, 96, 40)])
@pytest.mark.parametrize("window", [0, 1, 37])
def test_ragged_rows(hip, heads, n_kv, hd, vd, dtype, window):
    """Prompts, chunks behind cached rows, single tokens and sessions without rows."""
    s = Setup(hip, heads, n_kv, hd, [(19, 19), (70, 1), (33, 0), (90, 21), (0, 0), (1, 1), (47, 2)], ps=16, vd=vd,
              dtype=dtype, seed=3 + window).fill().upload()
    sinks = 2 * s.randn(heads) if window else None
    s.attend(s.round(1.5 * s.randn(s.n, heads, hd)), window, sinks)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ps", [16, 32, 48, 128])
def test_long_rows_split(hip, dtype, ps):
    """One long session: its range is split over workgroups and joined."""
    s = Setup(hip, 8, 2, 64, [(1500, 1)], ps=ps, dtype=dtype, seed=ps).fill().upload()
    q = s.round(1.5 * s.randn(1, 8, 64))
    assert s.workspace(1) is not None
    s.attend(q)
    s.attend(q, 700, 2 * s.randn(8))


@pytest.mark.parametrize("max_kv", [1, 100, 100000])
def test_any_length_hint_is_correct(hip, max_kv):
    s = Setup(hip, 4, 1, 128, [(700, 1), (3, 1), (260, 1)], ps=32, seed=5).fill().upload(max_kv=max_kv)
    s.attend(1.5 * s.randn(s.n, 4, 128))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [1e-4, 30.0])
def test_small_and_large_values(hip, dtype, scale):
    """Keys and values far from one, and scores that leave one key: maxima that
    grow along the row."""
    s = Setup(hip, 8, 2, 64, [(300, 1), (90, 3)], dtype=dtype, seed=9, scale=scale).fill().upload()
    s.attend(s.round(s.randn(s.n, 8, 64) * np.float32(1.0 if scale < 1 else 0.1)))


def test_rows_without_keys_are_zero(hip):
    """No page, a length of zero, fewer cached tokens than rows."""
    s = Setup(hip, 4, 2, 64, [(20, 1), (40, 3), (2, 2), (33, 1)], seed=11).fill().upload()
    s.table[0] = -1
    s.table[3, 0] = 10 ** 6  # a page id behind the pool: its positions are masked
    s.kv_lens[1] = 1         # rows at positions -2, -1, 0
    s.kv_lens[2] = 0
    s.upload()
    for sinks in (None, 2 * s.randn(4)):
        got = s.attend(s.randn(s.n, 4, 64), 0, sinks)
        assert (got[0] == 0).all() and (got[1:3] == 0).all() and (got[4:6] == 0).all()


def test_bad_pages_among_good_ones(hip):
    s = Setup(hip, 8, 2, 128, [(400, 1), (200, 5)], seed=12).fill()
    s.table[0, 3], s.table[0, 20], s.table[1, 0] = -1, s.pool.n_pages, -7
    s.upload()
    s.attend(1.5 * s.randn(s.n, 8, 128))
    s.attend(1.5 * s.randn(s.n, 8, 128), 100)


def test_table_shorter_than_the_length(hip):
    s = Setup(hip, 4, 1, 64, [(100, 2)], seed=13).fill()
    s.table = np.ascontiguousarray(s.table[:, :4])
    s.upload()
    s.attend(s.randn(s.n, 4, 64))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_nan_and_infinities_stay_out(hip, dtype):
    """Scales behind the last token, before the window and of later rows of the
    same chunk are NaN or infinite: no earlier row sees them."""
    import torch
    s = Setup(hip, 8, 2, 64, [(90, 9), (64, 1)], dtype=dtype, seed=14).fill()
    p = s.pool
    q = s.round(s.randn(s.n, 8, 64))
    for t, bits in ((89, 0x7E00), (88, 0x7C00), (2, 0xFC00)):
        page, off = s.table[0, t // p.ps], t % p.ps
        for h in range(p.n_kv):
            at = p._at(page, h) + p.ps * 16 * p.G + off * p.G * 2
            for buf in (p.k, p.v):
                buf[at:at + 2 * p.G].view(np.uint16)[:] = bits
    s.upload()
    # window 60: position 2 is out of sight of every row (81..89); rows 7 and 8 do
    # see positions 88 and 89, so only rows 0..6 and the other session are checked
    out = torch.zeros(s.n, 8, 64, dtype=_dtype(dtype), device=DEV)
    assert hip.paged_attention_dev(s.cache, s.batch, _t(q, _dtype(dtype)), out, 0.125, s.workspace(s.n), None, 60)
    got = out.float().cpu().numpy()
    assert np.isnan(got[8]).any() and np.isfinite(got[:7]).all() and np.isfinite(got[9]).all()
    for t in (88, 89):
        page, off = s.table[0, t // p.ps], t % p.ps
        p.store("k", page, off, s.randn(2, 64))
        p.store("v", page, off, s.randn(2, 64))
    ref, spread, size = R.attention(p, s.table, s.kv_lens, s.q_starts, q, 0.125, 60)
    tol = R.tolerance(ref, spread, size, dtype)
    rows = [0, 1, 2, 3, 4, 5, 6, 9]
    assert (np.abs(got - ref) <= tol)[rows].all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,n_kv,hd", [(16, 16, 64), (80, 16, 64), (128, 8, 64), (48, 16, 128), (8, 8, 256)])
def test_many_short_sessions(hip, heads, n_kv, hd, dtype):
    """Enough (session, kv head) pairs that each is one wave's: 1, 5, 16 and 3 query
    heads per kv head, with a window that cuts and sinks."""
    n = -(-2048 // n_kv)
    rng = np.random.default_rng(heads)
    lens = [int(x) for x in rng.integers(1, 19, n)]
    lens[:5] = [0, 40, 1, 70, 16]
    s = Setup(hip, heads, n_kv, hd, [(a, 1) for a in lens], dtype=dtype, seed=heads).fill().upload()
    q = s.round(1.5 * s.randn(s.n, heads, hd))
    assert s.workspace(s.n) is None  # nothing is split
    s.attend(q, 9, 2 * s.randn(heads))


def test_heads_that_do_not_share_evenly_are_refused(hip):
    """24 query heads of 16 kv heads, many sessions: no workspace and no call."""
    import torch
    s = Setup(hip, 24, 16, 128, [(16, 1)] * 128, seed=24).fill().upload()
    out = torch.full((s.n, 24, 128), 7.0, device=DEV)
    assert hip.paged_attention_workspace(s.cache, s.batch, s.n, 24) == 0
    assert not hip.paged_attention_dev(s.cache, s.batch, _t(s.randn(s.n, 24, 128)), out, 0.1, None, window=9)
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("sessions,most", [([(4928, 1), (70, 1), (4700, 1), (9, 1), (700, 1)], 4928),
                                           ([(3520, 100)], 3520)])
def test_windows_split_finer_than_the_whole_row(hip, sessions, most):
    """A window a little shorter than the context: its splits round to more than those
    of the whole row, for which the workspace is told."""
    import torch
    s = Setup(hip, 64, 8, 64, sessions, dtype="bf16", seed=most).fill().upload()
    q = s.round(s.randn(s.n, 64, 64))
    tq, ws = _t(q, torch.bfloat16), s.workspace(s.n)
    out = torch.empty_like(tq)
    for window in range(32, most, 32):
        assert hip.paged_attention_dev(s.cache, s.batch, tq, out, 0.125, ws, window=window), window
    for window in (most * 8 // 9, most - 40):
        s.attend(q, window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,n_kv,hd,window", [(8, 1, 64, 0), (4, 2, 128, 100), (5, 1, 128, 0), (2, 1, 256, 0),
                                                  (40, 2, 64, 0)])
def test_long_chunks(hip, heads, n_kv, hd, window, dtype):
    """Several tiles of one chunk, split over its cached rows, next to sessions of
    single tokens and a chunk of another length."""
    s = Setup(hip, heads, n_kv, hd, [(300, 1), (460, 71), (5, 1), (333, 33)], ps=32, dtype=dtype, seed=heads + hd).fill()
    s.upload()
    s.attend(s.round(1.5 * s.randn(s.n, heads, hd)), window, 2 * s.randn(heads) if window else None)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_scales_that_grow_and_shrink_along_the_row(hip, rows, dtype):
    """Values of 1e-4 at first, then 1, 300 and 1e-3: the common exponent follows the
    largest and nothing of the others is lost that matters."""
    s = Setup(hip, 8, 2, 64, [(400, rows)], dtype=dtype, seed=91)
    p = s.pool
    for t in range(400):
        size = np.float32([1e-4, 1.0, 300.0, 1e-3][t // 100])
        p.store("k", s.table[0, t // p.ps], t % p.ps, s.randn(2, 64))
        p.store("v", s.table[0, t // p.ps], t % p.ps, s.randn(2, 64) * size)
    s.upload()
    q = s.round(s.randn(rows, 8, 64))
    s.attend(q)
    s.kv_lens[0] = 110  # rows that see the small values and few of the next
    s.upload()
    s.attend(q)


@pytest.mark.parametrize("rows", [2, 40])
def test_nan_group_is_nan_where_it_is_seen(hip, rows):
    """One NaN scale of a value's second group: those 32 channels of the rows at and
    behind it, and nothing else."""
    import torch
    s = Setup(hip, 8, 2, 64, [(130, rows), (70, 1)], seed=92).fill()
    p = s.pool
    t = 130 - rows // 2 - 1  # inside the chunk
    page, off = s.table[0, t // p.ps], t % p.ps
    q = s.randn(s.n, 8, 64)
    ref, spread, size = R.attention(p, s.table, s.kv_lens, s.q_starts, q, 0.125)
    at = p._at(page, 1) + p.ps * 16 * p.G + (off * p.G + 1) * 2
    p.v[at:at + 2].view(np.uint16)[:] = 0x7E00
    s.upload()
    out = torch.zeros(s.n, 8, 64, device=DEV)
    assert hip.paged_attention_dev(s.cache, s.batch, _t(q), out, 0.125, s.workspace(s.n))
    got = out.cpu().numpy()
    want = np.zeros(got.shape, bool)
    sees = np.arange(s.n) >= rows - (130 - t)
    sees[rows:] = False
    want[sees, 4:, 32:] = True  # heads 4.. share kv head 1
    assert np.array_equal(np.isnan(got), want)
    assert (np.abs(got - ref) <= R.tolerance(ref, spread, size, "f32"))[~want].all()


NAN_SESSIONS = {  # kind: sessions, head dim, page size, heads
    "single": ([(1, 1), (70, 1), (2, 1)], 64, 16, 8),
    "split": ([(3000, 1), (1, 1), (900, 1)], 128, 64, 8),
    "one_wave_each": ([(1 + i % 19, 1) for i in range(1024)], 64, 16, 8),
    "chunk": ([(40, 40), (1, 1), (700, 60)], 64, 16, 8),
    "wide_chunk": ([(300, 40)], 128, 16, 8),
    "many_heads": ([(150, 3), (30, 20)], 64, 16, 40),
}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("kind", sorted(NAN_SESSIONS))
def test_nan_queries_and_seen_nan_keys_give_nan(hip, kind, sinks, dtype):
    """A NaN query, and a NaN key that a row sees, make all of that row's channels NaN
    (of the heads concerned), also where no other score is left, and no other row's."""
    import torch
    sessions, hd, ps, heads = NAN_SESSIONS[kind]
    s = Setup(hip, heads, 2, hd, sessions, ps=ps, dtype=dtype, seed=96).fill()
    q, sk = s.round(s.randn(s.n, heads, hd)), s.randn(heads) if sinks else None
    scale = np.float32(hd ** -0.5)
    ref, spread, size = R.attention(s.pool, s.table, s.kv_lens, s.q_starts, q, scale, 0, sk)
    tol = R.tolerance(ref, spread, size, dtype)
    want = np.zeros(ref.shape, bool)
    for row, head in ((0, 1), (s.n - 1, heads - 1), (s.n // 2, 0)):
        q[row, head, 3] = np.nan
        want[row, head] = True
    # the last session's key 0 of kv head 1, and the first session's last one of kv head 0
    p, mul, last = s.pool, heads // 2, len(sessions) - 1
    for seq, t, h in ((last, 0, 1), (0, int(s.kv_lens[0]) - 1, 0)):
        page, off = s.table[seq, t // p.ps], t % p.ps
        at = p._at(page, h) + p.ps * 16 * p.G + off * p.G * 2
        p.k[at:at + 2 * p.G].view(np.uint16)[:] = 0x7E00
        for r in range(s.q_starts[seq], s.q_starts[seq + 1]):
            if s.kv_lens[seq] - (s.q_starts[seq + 1] - r) >= t:
                want[r, h * mul:(h + 1) * mul] = True
    s.upload()
    out = torch.zeros(s.n, heads, hd, dtype=_dtype(dtype), device=DEV)
    assert hip.paged_attention_dev(s.cache, s.batch, _t(q, _dtype(dtype)), out, scale, s.workspace(s.n),
                                   None if sk is None else _t(sk))
    got = out.float().cpu().numpy()
    assert np.array_equal(np.isnan(got), want), np.argwhere(np.isnan(got) != want)[:4]
    assert (np.abs(got - ref) <= tol)[~want].all()


@pytest.mark.parametrize("scale", [-0.3, 0.0])
@pytest.mark.parametrize("rows", [1, 40])
def test_negative_and_zero_scale(hip, rows, scale):
    s = Setup(hip, 8, 2, 64, [(150, rows), (90, 1)], seed=93).fill().upload()
    s.attend(s.randn(s.n, 8, 64), scale=scale)


def test_rows_behind_the_last_session_are_left(hip):
    import torch
    s = Setup(hip, 4, 2, 64, [(20, 1), (300, 2)], seed=15).fill().upload()
    q = s.randn(s.n + 5, 4, 64)
    out = torch.full((s.n + 5, 4, 64), 7.0, device=DEV)
    assert hip.paged_attention_dev(s.cache, s.batch, _t(q), out, 0.125, s.workspace(s.n + 5))
    assert (out[s.n:] == 7.0).all() and (out[:s.n] != 7.0).all()


def test_more_rows_than_the_hint_are_left(hip):
    import torch
    s = Setup(hip, 4, 1, 64, [(600, 1), (500, 7)], seed=16).fill().upload(max_q=1)
    out = torch.full((s.n, 4, 64), 7.0, device=DEV)
    assert hip.paged_attention_dev(s.cache, s.batch, _t(s.randn(s.n, 4, 64)), out, 0.125, s.workspace(s.n))
    assert torch.isfinite(out).all() and (out[0] != 7.0).all() and (out[2:] == 7.0).all()


def test_strided_rows(hip):
    """q inside a fused q/k/v row, out inside a wider one."""
    import torch
    s = Setup(hip, 8, 2, 64, [(50, 3), (90, 1)], seed=17).fill().upload()
    q = 1.5 * s.randn(s.n, 8, 64)
    fused = torch.zeros(s.n, 12, 64, device=DEV)
    fused[:, :8] = _t(q)
    wide = torch.full((s.n, 9, 64), 7.0, device=DEV)
    assert hip.paged_attention_dev(s.cache, s.batch, fused[:, :8], wide[:, :8], 0.125, s.workspace(s.n))
    ref, spread, size = R.attention(s.pool, s.table, s.kv_lens, s.q_starts, q, 0.125)
    assert (np.abs(wide[:, :8].cpu().numpy() - ref) <= R.tolerance(ref, spread, size, "f32")).all()
    assert (wide[:, 8] == 7.0).all()


# ---- append and read ------------------------------------------------------------------
def _tables(hd, n, rot=None):
    ang = np.arange(n)[:, None] * (10000.0 ** (-np.arange(0, rot or hd, 2) / (rot or hd)))
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def _append(s, q, k, v, cos, sin, neox, rows=None, in_place=False):
    """Appends on the device and in the host pool; returns the device's queries."""
    import torch
    t = _dtype(s.dtype)
    tq = _t(q, t)
    q_out = tq if in_place else torch.full_like(tq, 7.0)
    assert s.hip.paged_append_dev(s.cache, s.batch, _t(k, t), _t(v, t), _t(cos), _t(sin), q=tq, q_out=q_out, neox=neox)
    want = np.full(q.shape, 7.0, np.float32) if not in_place else q.copy()
    p = s.pool
    for i in range(len(s.kv_lens)):
        a, b = int(s.q_starts[i]), int(s.q_starts[i + 1])
        for r in range(a, b):
            pos = int(s.kv_lens[i]) - (b - r)
            if pos < 0 or pos >= cos.shape[0]:
                continue
            want[r] = s.round(R.rotate(q[r], cos[pos], sin[pos], neox))
            if pos // p.ps >= s.table.shape[1] or not 0 <= s.table[i, pos // p.ps] < p.n_pages:
                continue
            p.store("k", s.table[i, pos // p.ps], pos % p.ps, R.rotate(k[r], cos[pos], sin[pos], neox))
            p.store("v", s.table[i, pos // p.ps], pos % p.ps, v[r])
    got = q_out.float().cpu().numpy()
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))
    for dev, host in ((s.k_dev, p.k), (s.v_dev, p.v)):
        diff = np.flatnonzero(dev.cpu().numpy() != host)
        assert diff.size == 0, (diff.size, diff[:8])
    return q_out


@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,n_kv,hd,vd", SHAPES[:-5] + [(3, 3, 96, 40), (8, 1, 192, 128), (10, 5, 112, 112)])
def test_append_is_the_definition(hip, heads, n_kv, hd, vd, dtype, neox):
    s = Setup(hip, heads, n_kv, hd, [(19, 19), (70, 1), (33, 0), (40, 7)], ps=16, vd=vd, dtype=dtype, seed=21).upload()
    cos, sin = _tables(hd, 80, hd // 16 * 16)
    q, k, v = (s.round(s.randn(s.n, *w)) for w in ((heads, hd), (n_kv, hd), (n_kv, vd)))
    _append(s, q, k, v, cos, sin, neox, in_place=neox)


@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("rot", [0, 16, 64])
def test_append_partial_rotation(hip, rot, neox):
    s = Setup(hip, 4, 2, 128, [(30, 5), (5, 5)], ps=32, seed=22).upload()
    cos, sin = _tables(128, 40, rot) if rot else (np.zeros((40, 0), np.float32),) * 2
    q, k, v = s.randn(s.n, 4, 128), s.randn(s.n, 2, 128), s.randn(s.n, 2, 128)
    _append(s, q, k, v, cos, sin, neox)


def test_append_values_at_the_edges(hip):
    """Zeros, one value, ties of both signs, ties between codes, subnormal and
    overflowing scales, infinities and NaN."""
    s = Setup(hip, 1, 1, 64, [(16, 16)], seed=23).upload()
    v = s.randn(16, 1, 64)
    v[0] = 0.0
    v[1], v[1, 0, 5], v[1, 0, 40] = 0.0, 3.0, -3.0
    v[2, 0, :32] = np.where(np.arange(32) % 2, 1.0, -1.0)
    v[3, 0, :32] = (np.arange(32) - 16) * 0.5  # quotients on halves of a code
    v[4] *= np.float32(1e-7)
    v[5] *= np.float32(1e-30)
    v[6] *= np.float32(1e38)
    v[7, 0, 3], v[7, 0, 33] = np.inf, -np.inf
    v[8, 0, 9] = np.nan
    v[9] = np.float32(2.0 ** -149)
    v[10] = -v[10]
    v[11] = np.float32(65504.0)
    v[12] = -0.0
    v[13] *= np.float32(6e4)
    cos, sin = np.ones((16, 32), np.float32), np.zeros((16, 32), np.float32)
    k = v.copy()
    k[7, 0], k[8, 0] = 1.0, 2.0  # inf * 0 of the rotation is not what is tested here
    _append(s, s.randn(16, 1, 64), k, v, cos, sin, False)


def test_append_leaves_out_what_has_no_place(hip):
    """Pages out of the pool, positions behind the table's row, behind max_pos and
    below zero; the rest of the batch is stored."""
    s = Setup(hip, 2, 2, 64, [(40, 2), (33, 3), (60, 2), (2, 2), (20, 1)], seed=24)
    s.table[0, 2] = -1
    s.table[1, 2] = s.pool.n_pages
    s.kv_lens[3] = 1  # rows at -1 and 0
    s.kv_lens[4] = 10 ** 6
    s.upload()
    cos, sin = _tables(64, 59)  # the third session's last row is at 59
    _append(s, s.randn(s.n, 2, 64), s.randn(s.n, 2, 64), s.randn(s.n, 2, 64), cos, sin, True)


def test_append_far_positions_and_large_pools(hip):
    """A position near the end of a 128 K context, in pages whose bytes pass 2^32."""
    import torch
    n_pages, ps, n_kv, hd = 8000, 1024, 8, 128
    size = hip.paged_kv_bytes(n_pages, ps, n_kv, hd)
    assert size > 2 ** 32
    k_dev, v_dev = (torch.zeros(size, dtype=torch.uint8, device=DEV) for _ in range(2))
    cache = hip.PagedKv(k_dev, v_dev, n_pages, ps, n_kv, hd)
    table = np.full((2, 128), -1, np.int32)
    table[0] = n_pages - 1 - np.arange(128)
    table[1, 0] = 0
    lens = np.array([131071, 1], np.int32)
    batch = hip.PagedBatch(_t(table), _t(lens), _t(np.array([0, 1, 2], np.int32)), 1, 131071)
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((2, n, hd)).astype(np.float32) for n in (16, n_kv, n_kv))
    cos, sin = _tables(hd, 131072)
    q_out = torch.empty(2, 16, hd, device=DEV)
    assert hip.paged_append_dev(cache, batch, _t(k), _t(v), _t(cos), _t(sin), q=_t(q), q_out=q_out)
    k_out, v_out = torch.empty(2, n_kv, hd, device=DEV), torch.empty(2, n_kv, hd, device=DEV)
    assert hip.paged_read_dev(cache, batch, k_out, v_out)
    for r, pos in enumerate((131070, 0)):
        for x, got in ((R.rotate(k[r], cos[pos], sin[pos], False), k_out[r]), (v[r], v_out[r])):
            c, d = R.quantize(x.reshape(n_kv, 4, 32))
            want = ((c.astype(np.float32) - 8) * d.astype(np.float32)[..., None]).reshape(n_kv, hd)
            assert np.array_equal(got.cpu().numpy(), want)
        assert np.array_equal(q_out[r].cpu().numpy(), R.rotate(q[r], cos[pos], sin[pos], False))
    # attention over 131071 positions, all but the last all-zero: uniform but for one
    out = torch.empty(2, 16, hd, device=DEV)
    ws = torch.empty(hip.paged_attention_workspace(cache, batch, 2, 16), dtype=torch.uint8, device=DEV)
    assert hip.paged_attention_dev(cache, batch, q_out, out, hd ** -0.5, ws)
    kk, vv = k_out[0].double().cpu().numpy(), v_out[0].double().cpu().numpy()
    w = hd ** -0.5 * np.einsum("hd,hd->h", q_out[0].double().cpu().numpy(), np.repeat(kk, 2, 0))
    want = (np.exp(w) / (np.exp(w) + 131070))[:, None] * np.repeat(vv, 2, 0)
    got = out.double().cpu().numpy()
    assert np.abs(got[0] - want).max() <= 1e-4 * np.abs(want).max()
    assert np.abs(got[1] - np.repeat(v_out[1].double().cpu().numpy(), 2, 0)).max() <= 2.0 ** -16 * np.abs(got[1]).max()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,n_kv,hd,vd", [(4, 4, 64, 64), (8, 2, 128, 128), (4, 2, 256, 256), (3, 3, 96, 40),
                                              (2, 1, 8, 16), (2, 2, 40, 200)])
def test_read_is_the_definition(hip, heads, n_kv, hd, vd, dtype):
    import torch
    s = Setup(hip, heads, n_kv, hd, [(19, 19), (70, 1), (33, 0), (40, 7)], ps=16, vd=vd, dtype=dtype, seed=31).fill()
    s.table[1, 4] = -1  # the second session's row has no page: its output rows stay
    s.upload()
    n = s.n + 2
    k = torch.full((n, n_kv, hd), 7.0, dtype=_dtype(dtype), device=DEV)
    v = torch.full((n, n_kv, vd), 7.0, dtype=_dtype(dtype), device=DEV)
    assert hip.paged_read_dev(s.cache, s.batch, k, v)
    wk, wv = np.full((n, n_kv, hd), 7.0, np.float32), np.full((n, n_kv, vd), 7.0, np.float32)
    for i in range(4):
        for r in range(s.q_starts[i], s.q_starts[i + 1]):
            pos = s.kv_lens[i] - (s.q_starts[i + 1] - r)
            page = s.table[i, pos // 16]
            if page >= 0:
                wk[r] = s.round(s.pool.load("k", page, pos % 16))
                wv[r] = s.round(s.pool.load("v", page, pos % 16))
    assert np.array_equal(k.float().cpu().numpy(), wk) and np.array_equal(v.float().cpu().numpy(), wv)
    only = torch.full_like(v, 7.0)
    assert hip.paged_read_dev(s.cache, s.batch, v_out=only)
    assert torch.equal(only, v)


# ---- together ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sessions_step_by_step(hip, dtype):
    """Prompts of three sessions, then decode steps of all: append, then attention,
    against the host's pool after every step."""
    import torch
    heads, n_kv, hd, ps = 8, 2, 64, 16
    s = Setup(hip, heads, n_kv, hd, [(40, 21), (40, 9), (40, 33)], ps=ps, dtype=dtype, seed=41).upload()
    cos, sin = _tables(hd, 64)
    lens = np.array([21, 9, 33], np.int32)
    for step in range(4):
        new = lens if step == 0 else np.ones(3, np.int32)
        s.kv_lens = lens if step == 0 else s.kv_lens + 1
        s.q_starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        s.n = int(s.q_starts[-1])
        s.t_lens, s.t_starts = _t(s.kv_lens.astype(np.int32)), _t(s.q_starts)
        s.batch = hip.PagedBatch(s.t_table, s.t_lens, s.t_starts, int(new.max()), 64)
        q, k, v = (s.round(s.randn(s.n, n, hd)) for n in (heads, n_kv, n_kv))
        q_rot = _append(s, q, k, v, cos, sin, True).float().cpu().numpy()
        s.attend(q_rot, 0 if step % 2 else 24)


def _graph_setup(hip, seed):
    s = Setup(hip, 8, 2, 64, [(600, 1), (90, 1), (300, 1)], dtype="bf16", seed=seed).fill().upload()
    cos, sin = (_t(a) for a in _tables(64, 700))
    import torch
    b = torch.bfloat16
    q, k, v = (_t(s.randn(3, n, 64), b) for n in (8, 2, 2))
    return s, cos, sin, q, k, v


def test_captured_and_replayed(hip):
    """append + attention in one graph, replayed over changing lengths, with eager
    calls in between on the same buffers."""
    import torch
    s, cos, sin, q, k, v = _graph_setup(hip, 51)
    q_rot, out, ws = torch.empty_like(q), torch.empty_like(q), s.workspace(3)

    def step():
        assert hip.paged_append_dev(s.cache, s.batch, k, v, cos, sin, q=q, q_out=q_rot)
        assert hip.paged_attention_dev(s.cache, s.batch, q_rot, out, 0.125, ws)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    start = torch.tensor([560, 50, 250], dtype=torch.int32, device=DEV)
    for i in range(4):
        s.t_lens.copy_(start + 9 * i)
        q.copy_(torch.randn_like(q))
        k.copy_(torch.randn_like(k))
        graph.replay()
        torch.cuda.synchronize()
        got, pools = out.clone(), (s.k_dev.clone(), s.v_dev.clone())
        out.fill_(7.0)
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, got) and torch.equal(s.k_dev, pools[0]) and torch.equal(s.v_dev, pools[1])


def test_a_captured_chunk(hip):
    """A prompt's chunk and decoding sessions in one graph, replayed over other
    queries and lengths."""
    import torch
    s = Setup(hip, 8, 2, 64, [(300, 60), (90, 1), (400, 1)], dtype="bf16", seed=94).fill().upload()
    q = _t(s.randn(s.n, 8, 64), torch.bfloat16)
    out, ws = torch.empty_like(q), s.workspace(s.n)
    call = lambda: hip.paged_attention_dev(s.cache, s.batch, q, out, 0.125, ws)  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call()
    start = torch.tensor([250, 40, 350], dtype=torch.int32, device=DEV)
    for i in range(3):
        s.t_lens.copy_(start + 17 * i)
        q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.fill_(7.0)
        assert call()
        torch.cuda.synchronize()
        assert torch.equal(out, got)


def test_the_current_device_and_stream_are_the_callers(hip):
    """A call on a stream given by handle, and torch's current device as it was."""
    import torch
    s = Setup(hip, 4, 2, 64, [(90, 1), (20, 2)], seed=95).fill().upload()
    q, st = s.randn(3, 4, 64), torch.cuda.Stream()
    tq, out, ws = _t(q), torch.zeros(3, 4, 64, device=DEV), s.workspace(3)
    torch.cuda.synchronize()
    assert hip.paged_attention_dev(s.cache, s.batch, tq, out, 0.125, ws, stream=st.cuda_stream)
    st.synchronize()
    assert torch.cuda.current_device() == 0
    ref, spread, size = R.attention(s.pool, s.table, s.kv_lens, s.q_starts, q, 0.125)
    assert (np.abs(out.cpu().numpy() - ref) <= R.tolerance(ref, spread, size, "f32")).all()


def test_two_streams_at_once(hip):
    """The same step of two caches on two streams, each after a long kernel on its
    own stream that writes its inputs: the calls wait for their stream alone."""
    import torch
    sets = [_graph_setup(hip, 61), _graph_setup(hip, 62)]
    want, got = [], []
    for s, cos, sin, q, k, v in sets:
        out, q_rot = torch.empty_like(q), torch.empty_like(q)
        assert hip.paged_append_dev(s.cache, s.batch, k, v, cos, sin, q=q, q_out=q_rot)
        assert hip.paged_attention_dev(s.cache, s.batch, q_rot, out, 0.125, s.workspace(3))
        want.append(out)
    big = torch.randn(4096, 4096, device=DEV)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    keep = []
    for st, (s, cos, sin, q, k, v) in zip(streams, sets):
        with torch.cuda.stream(st):
            x = big
            for _ in range(4):
                x = x @ big
            q2 = q + (x[0, 0] * 0).nan_to_num(0.0).to(q.dtype)
            out, q_rot, ws = torch.empty_like(q), torch.empty_like(q), s.workspace(3)
            assert hip.paged_append_dev(s.cache, s.batch, k, v, cos, sin, q=q2, q_out=q_rot)
            assert hip.paged_attention_dev(s.cache, s.batch, q_rot, out, 0.125, ws)
            got.append(out)
            keep += [x, q2, q_rot, ws]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_same_call_twice_gives_the_same_bits(hip):
    import torch
    s = Setup(hip, 8, 2, 128, [(900, 1), (700, 40), (65, 1)], seed=71).fill().upload()
    q = _t(1.5 * s.randn(s.n, 8, 128))
    outs = []
    for _ in range(3):
        out = torch.empty(s.n, 8, 128, device=DEV)
        assert hip.paged_attention_dev(s.cache, s.batch, q, out, 0.088, s.workspace(s.n))
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- refusals -----------------------------------------------------------------------------
def test_refusals(hip):
    import torch
    s = Setup(hip, 4, 2, 64, [(700, 1), (90, 2)], seed=81).fill().upload()
    q, out = _t(s.randn(3, 4, 64)), torch.full((3, 4, 64), 7.0, device=DEV)
    ws = s.workspace(3)
    with pytest.raises(ValueError):
        hip.paged_attention_dev(s.cache, s.batch, q.half(), out, 0.125, ws)
    with pytest.raises(ValueError):
        hip.paged_attention_dev(s.cache, s.batch, q, out.bfloat16(), 0.125, ws)
    with pytest.raises(ValueError):
        hip.paged_attention_dev(s.cache, s.batch, q, out[:, :, :32], 0.125, ws)
    with pytest.raises(ValueError):
        hip.paged_attention_dev(s.cache, s.batch, q.cpu(), out, 0.125, ws)
    assert not hip.paged_attention_dev(s.cache, s.batch, q[:, :3], out[:, :3], 0.125, ws)  # 3 heads of 2 kv heads
    assert not hip.paged_attention_dev(s.cache, s.batch, q, out, 0.125, None)
    assert not hip.paged_attention_dev(s.cache, s.batch, q, out, 0.125, ws[:-16])
    assert not hip.paged_attention_dev(s.cache, s.batch, q, out, float("nan"), ws)
    wide = torch.zeros(3 * 4 * 64 + 1, device=DEV)[1:].view(3, 4, 64)  # not aligned to four elements
    assert not hip.paged_attention_dev(s.cache, s.batch, wide, out, 0.125, ws)
    cos, sin = (_t(a) for a in _tables(64, 800))
    k, v = _t(s.randn(3, 2, 64)), _t(s.randn(3, 2, 64))
    with pytest.raises(ValueError):
        hip.paged_append_dev(s.cache, s.batch, k, v, cos, sin, q=q)
    with pytest.raises(ValueError):
        hip.paged_append_dev(s.cache, s.batch, k, v[:2], cos, sin)
    assert not hip.paged_append_dev(s.cache, s.batch, k, v, cos[:, :20].contiguous(), sin[:, :20].contiguous())
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    assert np.array_equal(s.k_dev.cpu().numpy(), s.pool.k) and np.array_equal(s.v_dev.cpu().numpy(), s.pool.v)
