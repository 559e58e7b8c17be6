"""Codes drawn from logits (qinco_amd.sample) and rows grouped by inverted list (qinco_amd.lists) against plain statements of both in 64
bits; their refusals; and a run of them together with the look-up decoder and the k-nearest-list search."""
import ctypes as C
import math

import numpy as np
import pytest

gpu = pytest.mark.gpu
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}   # half a step relative to the value


# ------------------------------------------------------------------------------------------------ plain statements
def draw_codes(z, u, T, k, p, m):
    """z (n, V) float64; settings per row.  -> codes, log probabilities in 64 bits."""
    n, V = z.shape
    codes, logps = np.full(n, -1, np.int64), np.full(n, -np.inf)
    T, k, p, m = (np.broadcast_to(np.asarray(v, np.float64), (n,)) for v in (T, k, p, m))
    for r in range(n):
        at = np.flatnonzero(z[r] > -np.inf)        # (NaN compares false)
        if not len(at):
            continue
        at = at[np.argsort(-z[r][at], kind="stable")]
        if T[r] <= 0:
            codes[r], logps[r] = at[0], 0.0
            continue
        if 0 < k[r] < V:
            at = at[: int(k[r])]
        top = z[r][at[0]]
        with np.errstate(invalid="ignore", over="ignore"):
            e = np.where(z[r][at] == top, 1.0, np.exp((z[r][at] - top) / T[r]))
        mass = np.cumsum(e)
        if p[r] < 1:
            before = np.concatenate([[0.0], mass[:-1]])
            stay = before < p[r] * mass[-1]
            stay[0] = True
            at, e = at[stay], e[stay]
        at, e = at[e >= min(m[r], 1.0)], e[e >= min(m[r], 1.0)]
        back = np.argsort(at)
        at, e = at[back], e[back]
        mass = np.cumsum(e)
        i = min(int(np.searchsorted(mass, min(max(u[r], 0.0), 1.0) * mass[-1], side="right")), int(np.flatnonzero(e).max()))
        codes[r], logps[r] = at[i], np.log(e[i] / mass[-1])
    return codes, logps


def sort_entries(ids, E):
    """ids (n, k) -> order, place, offsets by definition."""
    flat = np.asarray(ids).astype(np.int64).reshape(-1)
    entries = np.flatnonzero((flat >= 0) & (flat < E))
    entries = entries[np.argsort(flat[entries], kind="stable")]
    order, place = np.full(flat.size, -1, np.int64), np.full(flat.size, -1, np.int64)
    order[: len(entries)] = entries
    place[entries] = np.arange(len(entries))
    return order, place.reshape(np.shape(ids)), np.searchsorted(flat[entries], np.arange(E + 1))


def to64(t):
    return t.detach().double().cpu().numpy()


# ------------------------------------------------------------------------------------------------ CPU: refusals, sizes
@pytest.fixture(scope="module")
def lib():
    from qinco_amd import _lib, build
    build.build()
    return _lib.load()


def test_sample_refusals_are_decided_on_the_host(lib):
    from qinco_amd import _lib
    P = _lib.QincoSampleParams
    buf = (C.c_char * 64)()
    at = C.addressof(buf)

    def call(dtype=0, stride=8, n=1, V=8, params=None, codes=0, logits=at, u=at, out=at):
        params = P(struct_bytes=C.sizeof(P), temperature=1.0, top_p=1.0) if params is None else params
        return lib.qinco_sample_codes(logits, dtype, stride, n, V, u, 0, C.byref(params), out, codes, None, None, 0, None)
    assert call(n=0) == 0                                        # nothing to do: no launch
    for bad in (dict(dtype=3), dict(V=0), dict(V=(1 << 24) + 1), dict(n=-1), dict(n=1 << 31), dict(stride=-1), dict(codes=_lib.CODE_U8),
                dict(logits=None), dict(u=None), dict(out=None), dict(params=P(struct_bytes=8))):
        assert call(**bad) == -1, bad
        assert b"qinco_sample_codes" in lib.qinco_last_error()
    assert lib.qinco_sample_workspace(-1, 8) == 0 and lib.qinco_sample_workspace(4, 0) == 0
    assert lib.qinco_sample_codes(at, 0, 8, 1, 8, at, 0, None, at, 0, None, None, 0, None) == -1


def test_group_refusals_are_decided_on_the_host(lib):
    buf = (C.c_char * 64)()
    at = C.addressof(buf)

    def call(code=0, stride=1, n=4, k=1, E=8, lists=at, order=at, place=at, offsets=at, ws=at, ws_bytes=1 << 30):
        return lib.qinco_group_rows(lists, code, stride, n, k, E, order, place, offsets, None, ws, ws_bytes, None)
    for bad in (dict(code=3), dict(n=-1), dict(k=0), dict(n=1 << 30, k=4), dict(E=0), dict(E=(1 << 24) + 1), dict(stride=-1), dict(lists=None),
                dict(order=None), dict(place=None), dict(offsets=None), dict(ws=None), dict(ws_bytes=8)):
        assert call(**bad) == -1, bad
        assert b"qinco_group_rows" in lib.qinco_last_error()
    assert lib.qinco_group_workspace(-1, 8) == 0 and lib.qinco_group_workspace(4, 0) == 0 and lib.qinco_group_workspace(4, 1 << 25) == 0
    assert lib.qinco_group_workspace(0, 1) > 0

    def gather(x=at, xs=4, rb=4, order=at, place=at, end=at, n=2, k=2, out=at):
        return lib.qinco_group_gather(x, xs, rb, order, place, end, n, k, out, None)
    assert gather(n=0) == 0
    for bad in (dict(x=None), dict(xs=-1), dict(rb=0), dict(rb=1 << 31), dict(order=None), dict(place=None), dict(end=None), dict(n=-1), dict(k=0), dict(out=None),
                dict(n=1 << 30, k=2)):
        assert gather(**bad) == -1, bad

    def combine(y=at, dt=0, ys=4, D=4, w=at, wdt=0, place=at, n=2, k=2, out=at):
        return lib.qinco_group_combine(y, dt, ys, D, w, wdt, place, n, k, out, None)
    assert combine(n=0) == 0
    for bad in (dict(y=None), dict(dt=5), dict(ys=-1), dict(D=0), dict(wdt=1), dict(dt=1, wdt=2), dict(place=None), dict(n=-1), dict(k=0),
                dict(out=None)):
        assert combine(**bad) == -1, bad

    def grad(d=at, ds=4, y=at, ys=4, dt=0, D=4, w=at, wdt=0, place=at, end=at, n=2, k=2, dy=at, dw=at):
        return lib.qinco_group_combine_grad(d, ds, y, ys, dt, D, w, wdt, place, end, n, k, dy, dw, None)
    assert grad(n=0) == 0
    for bad in (dict(d=None), dict(ds=-1), dict(y=None), dict(ys=-1), dict(dt=3), dict(D=0), dict(w=None), dict(wdt=2), dict(place=None),
                dict(end=None), dict(n=-1), dict(k=0), dict(dy=None, dw=None)):
        assert grad(**bad) == -1, bad


def test_host_tensors_are_refused():
    import torch
    from qinco_amd import RowGroups, group_rows, sample_codes
    with pytest.raises(ValueError, match="logits must be a torch CUDA tensor"):
        sample_codes(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(ValueError, match="lists must be a torch CUDA tensor"):
        group_rows(torch.zeros(4, dtype=torch.int64), 8)
    with pytest.raises(ValueError, match="order must be a torch CUDA tensor"):
        RowGroups(*(torch.zeros(s, dtype=torch.int32) for s in ((4,), (4, 1), (9,))))


# ------------------------------------------------------------------------------------------------ sampling
def check_sample(z, u, *, T=1.0, k=0, p=1.0, m=0.0, code_dtype=np.int64):
    """z: CUDA (n, V); settings numbers or numpy arrays (n,).  The drawn codes equal the plain statement's; the log probabilities are
    theirs within the rounding to 32 bits (the 64-bit value itself is good to V 2^-42 of the mass)."""
    import torch
    from qinco_amd import sample_codes
    rows = {}
    for name, v, dt in (("temperature", T, torch.float32), ("top_k", k, torch.int32), ("top_p", p, torch.float32), ("min_p", m, torch.float32)):
        rows[name] = torch.as_tensor(v).to("cuda", dt) if isinstance(v, np.ndarray) else v
    codes, logp = sample_codes(z, u, code_dtype=code_dtype, return_logp=True, **rows)
    assert codes.dtype == (torch.int64 if code_dtype is np.int64 else torch.int32) and logp.dtype == torch.float32
    plain = [to64(v) if torch.is_tensor(v) else v for v in rows.values()]
    want, want_logp = draw_codes(to64(z), to64(u), *plain)
    got = codes.cpu().numpy()
    assert np.array_equal(got, want), (np.flatnonzero(got != want)[:5], got[got != want][:5], want[got != want][:5])
    gl, fin = to64(logp), np.isfinite(want_logp)
    assert np.array_equal(gl[~fin], want_logp[~fin])
    assert np.all(np.abs(gl[fin] - want_logp[fin]) <= 2.0 ** -24 * np.abs(want_logp[fin]) + z.shape[1] * 2.0 ** -42 + 1e-12)
    return codes


SETTINGS = [dict(), dict(T=0.7, k=5), dict(p=0.9), dict(m=0.05), dict(T=1.3, k=50, p=0.8, m=0.01), dict(T=0.0), dict(k=1), dict(p=0.0), dict(m=1.0),
            dict(p=1e-6), dict(T=1e-3, k=3, p=0.99), dict(T=1e-30, p=0.9), dict(T=1e30, p=0.5), dict(T=1e30, k=7, m=1.0)]


@gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,V", [(1, 1), (3, 2), (5, 63), (4, 64), (4, 65), (300, 256), (7, 257), (9, 512), (9, 513), (3, 1000), (5, 1024), (5, 1025), (6, 4099),
                                 (2, 2048), (2, 6145), (2, 10240), (2, 10241), (2, 16385), (2, 20480), (2, 20481), (2, 32769), (2, 70001), (1, (1 << 20) + 3),
                                 (2500, 100), (2500, 128), (2500, 200), (2500, 256), (257, 1025), (257, 2049), (257, 5121), (257, 10241)])
def test_sample_sizes_and_settings(dtype, n, V):
    import torch
    g = torch.Generator("cuda").manual_seed(n * 1000003 + V)
    for i, s in enumerate(SETTINGS if n * V < 100000 else SETTINGS[:5]):
        z = (torch.randn(n, V, generator=g, device="cuda") * 2.5).to(getattr(torch, dtype))
        check_sample(z, torch.rand(n, generator=g, device="cuda"), **s)


@gpu
def test_sample_masks_infinities_nan_and_ties():
    import torch
    g = torch.Generator("cuda").manual_seed(5)
    inf, low = float("inf"), torch.finfo(torch.float32).min
    for V, rep in ((2, 1), (64, 1), (100, 1), (100, 52), (200, 1), (200, 52), (256, 1), (500, 1), (900, 1), (1500, 1), (1500, 7), (4000, 7), (5001, 1), (6000, 7), (11000, 1), (40000, 1)):
        z = torch.randn(40, V, generator=g, device="cuda")
        z[0] = -inf                                    # nothing left
        z[1] = float("nan")
        z[2] = low                                     # the type's lowest value everywhere: a uniform row
        z[3] = low
        z[3, V // 2] = 0.0                             # ... everywhere but at one place
        z[4] = -inf
        z[4, V - 1] = -7.0                             # one code left
        z[5, ::2] = float("nan")
        z[6, 1::2] = -inf
        z[7, V // 2] = inf                             # all the mass at infinity, once
        z[8] = inf                                     # ... and everywhere
        z[9] = 0.0
        z[9, ::2] = -0.0                               # equal logits: -0 is 0
        z[10] = torch.randint(0, 3, (V,), generator=g, device="cuda").float()      # ties everywhere
        z[11] = 3e38
        z[11, 0] = -3e38
        z[12] = torch.randint(0, 100, (V,), generator=g, device="cuda") * 1.4e-45  # denormal logits
        z[13] = -inf
        z[13, 0] = low
        z[14] = torch.arange(V, device="cuda").float()
        z[15] = -torch.arange(V, device="cuda").float()
        z[16:24] = torch.randint(-2, 3, (8, V), generator=g, device="cuda").float()
        z[24:28, : V // 2] = -inf
        z = z.repeat(rep, 1)                           # (more rows than a card has CUs go another way)
        for s in SETTINGS if rep == 1 else SETTINGS[:5]:
            u = torch.rand(40 * rep, generator=g, device="cuda")
            u[20:24] = torch.tensor([0.0, 1.0 - 2.0 ** -24, 0.5, 2.0 ** -30])
            check_sample(z, u, **s)


@gpu
@pytest.mark.parametrize("V", [40, 200, 500, 1000, 6000, 20000])
def test_sample_temperatures_whose_reciprocal_overflows(V):
    """1 / T is infinite: the largest logits share all the mass, wherever the cuts are."""
    import torch
    g = torch.Generator("cuda").manual_seed(V)
    z = torch.randn(6, V, generator=g, device="cuda")
    z[2:4] = torch.randint(-2, 3, (2, V), generator=g, device="cuda").float()
    z[4, ::2] = -float("inf")
    z[5] = 0.25
    u = torch.tensor([0.0, 0.9, 0.3, 0.999, 0.5, 0.7], device="cuda")
    for T in (1e-310, 5e-324, 2.3e-308, np.full(6, 1e-45, np.float32)):
        for s in (dict(), dict(p=0.5), dict(k=3), dict(k=30, p=0.3), dict(m=0.5)):
            check_sample(z, u, T=T, **s)


@gpu
def test_sample_borders_fall_on_the_exact_side():
    """256 equal logits: the running mass passes u = j / 256 only behind code j; a distribution drawn at evenly spaced numbers has every
    code as often as its mass says, to within one."""
    import torch
    from qinco_amd import sample_codes
    for dt in (torch.float64, torch.float32):
        u = torch.arange(256, device="cuda", dtype=dt) / 256
        got = sample_codes(torch.zeros(256, 256, device="cuda"), u)
        assert got.tolist() == list(range(256))
    assert sample_codes(torch.zeros(5, 256, device="cuda"), torch.tensor([-1.0, float("nan"), 1.0, 7.0, float("inf")], device="cuda")).tolist() == [0, 0, 255, 255, 255]
    n = 20000
    z = torch.randn(1, 100, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    got = np.bincount(sample_codes(z.expand(n, 100), (torch.arange(n, device="cuda", dtype=torch.float64) + 0.5) / n).cpu().numpy(), minlength=100)
    e = np.exp(to64(z)[0] - to64(z).max())
    assert np.all(np.abs(got - n * e / e.sum()) <= 1.0)


def hard_rows(V, g):
    """Rows whose cuts fall among many codes: few values, values that hardly differ, far outliers, long tails."""
    import torch
    rand = lambda: torch.rand(V, generator=g, device="cuda")               # noqa: E731
    low = torch.finfo(torch.float32).min
    near, small = 1.0 + rand() * 1e-3, rand() * 1e-4
    masked = near.clone()
    masked[rand() < 0.5] = low
    apart = small.clone()
    apart[V // 3] = -50.0                                                  # all the others in one bin, all different
    steps = (rand() * 4).floor()
    clusters = torch.where(rand() < 0.5, rand() * 1e-5, 5.0 + rand() * 1e-5)
    return torch.stack([torch.zeros(V, device="cuda"), steps, near, masked, apart, clusters, -torch.exp(rand() * 30 - 15), rand().log(),
                        torch.full((V,), low, device="cuda"), (rand() * 1e6).floor() * 1e-3])


@gpu
@pytest.mark.parametrize("V", [60, 200, 500, 1024, 2000, 3000, 10240, 20480, 70001, 300001])
def test_sample_rows_that_pile_up_in_a_few_bins(V):
    import torch
    g = torch.Generator("cuda").manual_seed(V)
    z = hard_rows(V, g)
    for s in (dict(p=0.5), dict(k=V // 3), dict(k=V // 2, p=0.7), dict(k=V // 2, p=0.7, m=0.999, T=0.3), dict(m=0.9995), dict(T=100.0, p=0.3), dict(T=1e-3, p=0.99)):
        check_sample(z, torch.rand(len(z), generator=g, device="cuda", dtype=torch.float64), **s)


@gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_sample_long_rows_of_few_values(dtype):
    import torch
    g = torch.Generator("cuda").manual_seed(1)
    z = (torch.randn(3, 1 << 20, generator=g, device="cuda") * 2.5).to(getattr(torch, dtype))
    for s in (dict(p=0.9), dict(k=20000, p=0.5, m=1e-4), dict(T=3.0, p=0.99)):
        check_sample(z, torch.rand(3, generator=g, device="cuda"), **s)


@gpu
def test_sample_settings_per_row_strides_and_types():
    import torch
    from qinco_amd import sample_codes
    rs = np.random.RandomState(3)
    g = torch.Generator("cuda").manual_seed(3)
    for n, V in ((70, 256), (9, 3000), (3, 50001)):
        T = rs.uniform(0.2, 2, n).astype(np.float32)
        T[0], T[1] = 0.0, -1.0
        k = rs.randint(-1, 60, n).astype(np.int32)
        p = rs.uniform(0.1, 1.2, n).astype(np.float32)
        m = rs.uniform(-0.1, 0.3, n).astype(np.float32)
        wide = torch.randn(n, V + 7, generator=g, device="cuda") * 3
        z = wide[:, 3:3 + V]                                        # rows that start anywhere
        u = torch.rand(2 * n, generator=g, device="cuda", dtype=torch.float64)[::2]
        a = check_sample(z, u, T=T, k=k, p=p, m=m)
        b = check_sample(z.T.contiguous().T, u, T=T, k=k, p=p, m=m, code_dtype=np.int32)   # neighbouring codes far apart
        assert torch.equal(a, b.long())
        one = torch.cat([sample_codes(z[i:i + 1], u[i:i + 1], temperature=torch.from_numpy(T[i:i + 1]).cuda(),
                                      top_k=torch.from_numpy(k[i:i + 1]).cuda(), top_p=torch.from_numpy(p[i:i + 1]).cuda(),
                                      min_p=torch.from_numpy(m[i:i + 1]).cuda()) for i in range(n)])
        assert torch.equal(a, one)                                  # a row's code does not depend on its batch
    assert sample_codes(torch.zeros(0, 16, device="cuda"), torch.zeros(0, device="cuda")).shape == (0,)


@gpu
def test_sample_refuses():
    import torch
    from qinco_amd import sample_codes
    z, u = torch.zeros(4, 8, device="cuda"), torch.zeros(4, device="cuda")
    for bad in (dict(temperature=-1.0), dict(temperature=math.inf), dict(temperature=math.nan), dict(top_p=math.nan), dict(min_p=1.5),
                dict(code_dtype=np.uint8), dict(top_k=torch.zeros(4, device="cuda")), dict(top_p=torch.zeros(3, device="cuda")),
                dict(temperature=torch.ones(4)), dict(min_p=torch.zeros(4, device="cuda", dtype=torch.float64))):
        with pytest.raises(ValueError):
            sample_codes(z, u, **bad)
    for args in ((z[0], u), (z.long(), u), (z.double(), u), (z[:, :0], u), (z, u[:3]), (z, u.half()), (z, u.cpu())):
        with pytest.raises(ValueError):
            sample_codes(*args)


# ------------------------------------------------------------------------------------------------ grouping
def check_group(ids, E, **kw):
    from qinco_amd import group_rows
    g = group_rows(ids, E, **kw)
    order, place, offsets = sort_entries(ids.cpu().numpy() if ids.dim() == 2 else ids.cpu().numpy()[:, None], E)
    assert np.array_equal(g.order.cpu().numpy(), order)
    assert np.array_equal(g.place.cpu().numpy(), place)
    assert np.array_equal(g.offsets.cpu().numpy(), offsets)
    assert np.array_equal(g.counts().cpu().numpy(), np.diff(offsets))
    return g


@gpu
@pytest.mark.parametrize("N", [0, 1, 63, 64, 65, 511, 513, 4095, 4096, 4097, 8193, 20001, 100003])
def test_group_sizes(N):
    import torch
    g = torch.Generator("cuda").manual_seed(N)
    for E in (1, 2, 255, 256, 257, 2047, 2048, 2049, 4096, 4097, 65536, 1 << 20, (1 << 22) + 1, 1 << 24):
        if E > 1 << 20 and N not in (65, 4097, 100003):
            continue
        ids = torch.randint(0, E, (N,), generator=g, device="cuda")
        check_group(ids, E)
        if N:
            ids[torch.rand(N, generator=g, device="cuda") < 0.2] = -1 - E
            check_group(ids.int(), E)
    if N:
        check_group(torch.full((N,), 300, device="cuda"), 512)                       # one list takes all
        check_group(torch.full((N,), -1, device="cuda"), 70000)                      # nothing has a list
        check_group(torch.full((N,), 99999, device="cuda"), 100000)
        check_group(torch.arange(N, device="cuda").flip(0), N)
        check_group(torch.randint(0, 256, (N,), generator=g, device="cuda").to(torch.uint8), 256)


@gpu
@pytest.mark.parametrize("N", [300001, 700001, 2100003])
def test_group_many_entries(N):
    import torch
    g = torch.Generator("cuda").manual_seed(N)
    for E in (1000, 70000, 1 << 20, 1 << 24):
        r = torch.rand(N, generator=g, device="cuda", dtype=torch.float64)
        ids = (r.pow(8) * E).long().clamp_(max=E - 1)                                # half of them in a few lists
        ids[torch.rand(N, generator=g, device="cuda") < 0.1] = -1
        check_group(ids, E, check=False)
    check_group(torch.full((N,), 70001, device="cuda", dtype=torch.int32), 1 << 17)
    check_group(torch.where(torch.arange(N, device="cuda") % 3 == 0, 5, 131000), 1 << 17)


@gpu
def test_group_matrices_columns_and_bad_ids():
    import torch
    from qinco_amd import group_rows
    g = torch.Generator("cuda").manual_seed(2)
    for n, k, E in ((1, 1, 1), (7, 3, 5), (1000, 8, 1024), (2049, 16, 77), (30000, 5, 1 << 18)):
        ids = torch.randint(-1, E, (n, k), generator=g, device="cuda")
        check_group(ids, E)
        wide = torch.randint(0, E, (n, k + 4), generator=g, device="cuda")
        check_group(wide[:, 2:2 + k], E)                                             # rows further apart than their ids
        check_group(wide[:, 1], E)                                                   # a column of a code matrix
        check_group(wide[:, ::2], E)
        check_group(wide[:1].expand(n, -1), E)
    ids = torch.tensor([[0, 5], [9, -1], [1 << 40, 2]], device="cuda")
    with pytest.raises(IndexError, match="n_lists"):
        group_rows(ids, 9)
    check_group(ids, 9, check=False)                                                 # ... or counts as having no list
    for args in ((ids.float(), 9), (ids, 0), (ids, (1 << 24) + 1), (ids[None], 9), (ids[:, :0], 9), (ids.cpu(), 9)):
        with pytest.raises(ValueError):
            group_rows(*args)


def make_groups(g, n, k, E, drop):
    import torch
    ids = torch.randint(0, E, (n, k), generator=g, device="cuda")
    if drop:
        ids[torch.rand(n, k, generator=g, device="cuda") < 0.3] = -1
        ids[n // 2] = -1                                                             # a row without any list
    from qinco_amd import group_rows
    return group_rows(ids, E)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,k,D", [(1, 1, 1), (5, 1, 3), (33, 2, 8), (64, 3, 96), (100, 8, 128), (77, 9, 101), (300, 16, 100), (50, 4, 768),
                                   (20, 17, 1023), (3000, 2, 256), (9, 33, 2)])
def test_gather_and_combine_with_gradients(dtype, n, k, D):
    """Against the formulas in 64 bits.  A sum of k products in 32 bits, in order: (k + 1) 2^-24 of the sum of absolute products; a dot
    product of D: D 2^-24 of the same; a product: 2^-24 of itself; and half a step of the type at the end (for fp16 2^-25 below its
    normal range)."""
    import torch
    g = torch.Generator("cuda").manual_seed(n * 131 + k * 17 + D)
    dt, half = getattr(torch, dtype), HALF[dtype]
    tiny = 2.0 ** -25 if dtype == "float16" else 0.0
    for drop in (False, True):
        gr = make_groups(g, n, k, 50, drop)
        place = gr.place.cpu().numpy()
        used = place >= 0
        at = np.where(used, place, 0)
        x = torch.randn(n, D, generator=g, device="cuda").to(dt).requires_grad_()
        out = gr.gather(x)
        want = np.zeros((n * k, D))
        want[place[used]] = np.repeat(to64(x), k, 0)[used.reshape(-1)]
        assert np.array_equal(to64(out), want)
        dout = torch.randn(n * k, D, generator=g, device="cuda").to(dt)
        dx, = torch.autograd.grad(out, x, dout)
        terms = np.where(used[:, :, None], to64(dout)[at], 0.0)
        assert dx.dtype == dt and np.all(np.abs(to64(dx) - terms.sum(1)) <= (k + 1) * 2.0 ** -24 * np.abs(terms).sum(1) + half * np.abs(terms.sum(1)) + tiny)
        for wdt in {torch.float32, dt}:
            y = torch.randn(n * k, D, generator=g, device="cuda").to(dt)
            y[gr.order < 0] = float("nan")                                           # rows no entry owns: whatever was there
            w = torch.softmax(torch.randn(n, k, generator=g, device="cuda"), 1).to(wdt)
            w[gr.place < 0] = float("nan")
            y.requires_grad_(), w.requires_grad_()
            out = gr.combine(y, w)
            y64, w64 = np.where(used[:, :, None], to64(y)[at], 0.0), np.where(used, to64(w), 0.0)
            terms = w64[:, :, None] * y64
            assert out.dtype == dt and np.all(np.abs(to64(out) - terms.sum(1)) <= (k + 1) * 2.0 ** -24 * np.abs(terms).sum(1) + half * np.abs(terms.sum(1)) + tiny)
            d = torch.randn(n, D, generator=g, device="cuda").to(dt)
            dy, dw = torch.autograd.grad(out, (y, w), d, retain_graph=True)
            d64 = to64(d)
            want = np.zeros((n * k, D))
            want[place[used]] = (w64[:, :, None] * d64[:, None])[used]
            assert dy.dtype == dt and np.all(np.abs(to64(dy) - want) <= (half + 2.0 ** -24) * np.abs(want) * (1 + 2.0 ** -20) + tiny)
            terms = d64[:, None] * y64
            tol = D * 2.0 ** -24 * np.abs(terms).sum(2) + (HALF[str(wdt)[6:]] if wdt != torch.float32 else 2.0 ** -24) * np.abs(terms.sum(2)) + (2.0 ** -25 if wdt == torch.float16 else 0)
            assert dw.dtype == wdt and np.all(np.abs(to64(dw) - terms.sum(2)) <= tol)
            assert torch.equal(torch.autograd.grad(out, y, d, retain_graph=True)[0], dy) and torch.equal(torch.autograd.grad(out, w, d)[0], dw)
        y = torch.randn(n * k, D, generator=g, device="cuda").to(dt).requires_grad_()
        out = gr.combine(y)
        terms = np.where(used[:, :, None], to64(y)[at], 0.0)
        assert np.all(np.abs(to64(out) - terms.sum(1)) <= (k + 1) * 2.0 ** -24 * np.abs(terms).sum(1) + half * np.abs(terms.sum(1)) + tiny)
        dy, = torch.autograd.grad(out, y, d)
        want = np.zeros((n * k, D))
        want[place[used]] = np.repeat(d64, k, 0)[used.reshape(-1)]
        assert np.array_equal(to64(dy), want)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_infinities_in_the_overlap_of_the_last_unit(dtype):
    """A row's last 16 bytes overlap the ones before them: an infinity there is summed once, and times nothing else."""
    import torch
    g = torch.Generator("cuda").manual_seed(21)
    gr = make_groups(g, 40, 3, 10, False)
    for D in (9, 11, 13):
        y = torch.rand(120, D, generator=g, device="cuda") + 0.5
        y[::4, D - 3] = float("inf")
        y[1::4, D - 2] = -float("inf")
        y = y.to(getattr(torch, dtype))
        d = (torch.rand(40, D, generator=g, device="cuda") + 0.5).to(y.dtype)
        d[::5, D - 3] = float("inf")
        w = torch.rand(40, 3, generator=g, device="cuda").requires_grad_()
        dw, = torch.autograd.grad(gr.combine(y, w), w, d)
        with np.errstate(invalid="ignore"):
            want = (to64(d)[:, None] * to64(y)[gr.place.cpu().numpy()]).sum(2)
        got, fin = to64(dw), np.isfinite(want)
        assert np.array_equal(got[~fin], want[~fin], equal_nan=True) and 0 < fin.sum() < fin.size
        assert np.all(np.abs(got[fin] - want[fin]) <= (D + 1) * 2.0 ** -24 * want[fin])      # (all terms positive)


@gpu
def test_gradients_against_differences():
    """Both operators are linear in the rows and in the weights: the difference over a step of 1 along a direction is the gradient's
    product with it, up to the rounding of two sums of some thousand terms of size 1 in 32 bits."""
    import torch
    g = torch.Generator("cuda").manual_seed(8)
    gr = make_groups(g, 60, 4, 30, True)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")          # noqa: E731
    x, y, w, c, ck = rand(60, 40), rand(240, 40), rand(60, 4), rand(60, 40), rand(240, 40)
    for f, t in ((lambda v: (gr.gather(v).double() * ck).sum(), x), (lambda v: (gr.combine(v, w).double() * c).sum(), y),
                 (lambda v: (gr.combine(y, v).double() * c).sum(), w)):
        v = t.clone().requires_grad_()
        grad, = torch.autograd.grad(f(v), v)
        step = rand(*t.shape)
        diff = float(f(t + step) - f(t))
        assert abs(diff - float((grad.double() * step).sum())) <= 1e-2, diff


@gpu
def test_rows_of_any_type_stride_and_broadcast_gradients():
    import torch
    g = torch.Generator("cuda").manual_seed(4)
    n, k = 501, 3
    gr = make_groups(g, n, k, 40, True)
    order = gr.order.cpu().numpy()
    for dt in (torch.uint8, torch.int32, torch.int64, torch.float64, torch.bool):
        for D in (1, 2, 4, 7, 8, 9, 16, 33):
            x = torch.randint(0, 100, (n, D + 5), generator=g, device="cuda").to(dt)
            for v in (x[:, :D], x[:, 2:2 + D], x.T.contiguous().T[:, :D], x[:1, :D].expand(n, D)):
                got = gr.gather(v).cpu().numpy()
                want = np.where((order >= 0)[:, None], v.cpu().numpy()[order // k], np.zeros((), got.dtype))
                assert np.array_equal(got, want)
    y = torch.randn(n * k, 24, generator=g, device="cuda")
    w = torch.rand(n, k, generator=g, device="cuda")
    base = gr.combine(y[:, 3:19].contiguous(), w)
    assert torch.equal(gr.combine(y[:, 3:19], w), base)                              # rows off their natural alignment: the same bits
    assert torch.equal(gr.combine(y.T.contiguous().T[:, 3:19], w.T.contiguous().T), base)
    leaf = y.clone().requires_grad_()
    gr.combine(leaf[:, 3:19], w).sum().backward()                                    # a gradient broadcast from one number
    want = np.zeros((n * k, 24))
    want[:, 3:19] = np.where((order >= 0)[:, None], to64(w).reshape(-1)[order][:, None], 0.0)
    assert np.array_equal(to64(leaf.grad), want)
    x = torch.randn(n, 16, generator=g, device="cuda", requires_grad=True)
    gr.gather(x).sum().backward()
    assert np.array_equal(to64(x.grad), np.repeat((gr.place.cpu().numpy() >= 0).sum(1)[:, None], 16, 1))
    shared = torch.randn(1, 16, generator=g, device="cuda", requires_grad=True)      # one row for all
    gr.gather(shared.expand(n, 16)).sum().backward()
    assert np.array_equal(to64(shared.grad)[0], np.full(16, float((gr.place >= 0).sum())))
    with pytest.raises(ValueError):
        gr.gather(torch.randn(n, 4, device="cuda", dtype=torch.float64, requires_grad=True))
    for call in (lambda: gr.gather(x[:-1]), lambda: gr.gather(x[:, :0]), lambda: gr.gather(x.cpu()), lambda: gr.combine(y[:-1]),
                 lambda: gr.combine(y.double()), lambda: gr.combine(y, w[:-1]), lambda: gr.combine(y, w.half()), lambda: gr.combine(y, w.cpu())):
        with pytest.raises(ValueError):
            call()


@gpu
def test_views_that_torch_conjugates_or_negates_on_reading():
    import torch
    from qinco_amd import sample_codes
    g = torch.Generator("cuda").manual_seed(22)
    n, k = 30, 2
    gr = make_groups(g, n, k, 7, False)

    def minus(*shape):                                         # the negated imaginary part, a view that holds the positive one
        z = torch.complex(torch.zeros(shape, device="cuda"), torch.rand(shape, generator=g, device="cuda") + 0.5)
        v = z.conj().imag
        assert v.is_neg() and bool((v < 0).all())
        return v
    for D in (1, 6):
        y, w = minus(n * k, D), minus(n, k)
        assert torch.equal(gr.combine(y, w), gr.combine(y.clone(), w.clone())) and bool((gr.combine(y, w) > 0).all())
        x = minus(n, D)
        assert torch.equal(gr.gather(x), gr.gather(x.clone()))
        c = torch.randn(n, D, generator=g, device="cuda", dtype=torch.complex64).conj()
        assert c.is_conj() and torch.equal(gr.gather(c), c[gr.order.long() // k])
    leaf = torch.rand(n, 1, generator=g, device="cuda").requires_grad_()
    gr.gather(leaf).backward(minus(n * k, 1))
    assert bool((leaf.grad < 0).all())
    z = minus(1, 1)
    assert torch.equal(sample_codes(z.expand(4, 1), torch.rand(4, device="cuda")), torch.zeros(4, dtype=torch.int64, device="cuda"))
    z = torch.cat([minus(4, 5), torch.zeros(4, 5, device="cuda")], 1)
    assert bool((sample_codes(z, torch.rand(4, device="cuda"), temperature=0.0) == 5).all())
    z = minus(4, 5)
    assert torch.equal(sample_codes(z, torch.rand(4, device="cuda"), temperature=0.0), z.argmax(1))


@gpu
def test_rows_too_long_are_refused():
    import torch
    gr = make_groups(torch.Generator("cuda").manual_seed(1), 1, 1, 1, False)
    for f in (gr.gather, gr.combine):
        with pytest.raises(ValueError, match="2\\^31"):
            f(torch.zeros(1, 1, device="cuda").expand(1, (1 << 32) + 5))


@gpu
def test_second_derivatives_are_refused_and_first_ones_with_their_graph_are_not():
    import torch
    g = torch.Generator("cuda").manual_seed(5)
    gr = make_groups(g, 20, 2, 5, False)
    x, y = torch.randn(20, 8, device="cuda", requires_grad=True), torch.randn(40, 8, device="cuda", requires_grad=True)
    w = torch.rand(20, 2, device="cuda", requires_grad=True)
    for out, leaves in ((gr.gather(x), (x,)), (gr.combine(y, w), (y, w)), (gr.combine(y), (y,))):
        plain = torch.autograd.grad(out.square().sum(), leaves, retain_graph=True)
        grads = torch.autograd.grad(out.square().sum(), leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, grads))
        with pytest.raises(RuntimeError, match="once_differentiable"):
            grads[0].sum().backward()


@gpu
def test_places_that_cannot_be_are_not_followed():
    """RowGroups built from other tensors than group_rows made: a slot outside (n k,) counts as none."""
    import torch
    from qinco_amd import RowGroups
    n, k = 6, 2
    place = torch.tensor([[0, 1], [2, 12], [1 << 30, 3], [-7, 4], [5, -(1 << 31)], [6, 7]], dtype=torch.int32, device="cuda")
    gr = RowGroups(torch.arange(12, dtype=torch.int32, device="cuda"), place, torch.tensor([0, -5], dtype=torch.int32, device="cuda"))
    y = torch.arange(12.0, device="cuda")[:, None].expand(12, 20).contiguous()
    assert gr.combine(y)[:, 0].tolist() == [1.0, 2.0, 3.0, 4.0, 5.0, 13.0]
    assert gr.gather(torch.ones(n, 20, device="cuda")).shape == (12, 20)
    for bad in ((place[:, 0], place, place[:, 0]), (place.reshape(-1), place, place.reshape(-1)[:1]), (place.reshape(-1)[:-1], place, place.reshape(-1)),
                (place.reshape(-1).long(), place, place.reshape(-1)), (place.reshape(-1), place.T, place.reshape(-1))):
        with pytest.raises(ValueError):
            RowGroups(*bad)


@gpu
def test_rows_behind_four_giga_elements():
    """2.3 G elements of y and of the gathered rows: places behind 32 bits of element offsets."""
    import torch
    from qinco_amd import group_rows
    n, k, D = 1_150_000, 2, 1000
    ids = torch.stack([torch.arange(n, device="cuda"), torch.arange(n, device="cuda")], 1)          # row r in places 2 r, 2 r + 1
    gr = group_rows(ids, n)
    assert torch.equal(gr.order, torch.arange(n * k, dtype=torch.int32, device="cuda"))
    x = torch.randint(0, 256, (n, D), device="cuda", dtype=torch.uint8)
    out = gr.gather(x)
    for r in (0, 1, n // 2, n - 2, n - 1):
        assert torch.equal(out[2 * r], x[r]) and torch.equal(out[2 * r + 1], x[r])
    assert torch.equal(out[::2], x) and torch.equal(out[1::2], x)
    del x
    y = out.to(torch.bfloat16)
    del out
    w = torch.tensor([[1.0, -0.5]], device="cuda").expand(n, 2)
    got = gr.combine(y, w)
    assert torch.equal(got, y[::2] * 0.5)
    dy, dw = gr._combine_grad(got, y, w.contiguous(), True, True)
    assert torch.equal(dy[::2], got) and torch.equal(dy[1::2], got * -0.5)
    for r in (0, n // 2, n - 1):
        want = float((got[r].double() * y[2 * r].double()).sum())
        assert abs(float(dw[r, 0]) - want) <= D * 2.0 ** -24 * want and float(dw[r, 0]) == float(dw[r, 1])


@gpu
def test_no_rows():
    import torch
    from qinco_amd import group_rows
    gr = group_rows(torch.zeros(0, 3, dtype=torch.int64, device="cuda"), 17)
    assert gr.offsets.tolist() == [0] * 18
    x = torch.zeros(0, 5, device="cuda", requires_grad=True)
    out = gr.combine(gr.gather(x), torch.zeros(0, 3, device="cuda"))
    assert out.shape == (0, 5)
    out.sum().backward()
    assert x.grad.shape == (0, 5)


# ------------------------------------------------------------------------------------------------ streams, graphs, together
@gpu
def test_streams_and_two_calls_at_once():
    import torch
    from qinco_amd import group_rows, sample_codes
    g = torch.Generator("cuda").manual_seed(6)
    jobs = []
    for i, (n, V, E) in enumerate(((3000, 256, 1 << 20), (2, 300000, 700), (40, 5000, 5000))):
        z, u = torch.randn(n, V, generator=g, device="cuda") * 3, torch.rand(n, generator=g, device="cuda")
        ids = torch.randint(0, E, (20000 + i, 2), generator=g, device="cuda")
        jobs.append((z, u, ids, E))
    work = lambda z, u, ids, E: (sample_codes(z, u, top_k=100, top_p=0.9), *(lambda q: (q.order, q.place, q.offsets))(group_rows(ids, E, check=False)))  # noqa: E731
    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(work(*j))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


@gpu
def test_two_graphs_replay_the_eager_results():
    """Two captured runs of everything, replayed in turn with new inputs and eager work between them."""
    import torch
    from qinco_amd import group_rows, sample_codes
    g = torch.Generator("cuda").manual_seed(7)
    sizes = ((600, 256, 4, 16), (5, 150000, 3, 100))

    def inputs(n, V, k, D):
        return (torch.randn(n, V, generator=g, device="cuda") * 2, torch.rand(n, generator=g, device="cuda"),
                torch.randint(-1, 5000, (n * 50, k), generator=g, device="cuda"), torch.randn(n * 50, D, generator=g, device="cuda"))

    def work(z, u, ids, x):
        codes = sample_codes(z, u, top_k=40, top_p=0.9, min_p=0.001)
        gr = group_rows(ids, 5000, check=False)
        rows = gr.gather(x)
        return codes, gr.order, gr.offsets, rows, gr.combine(rows, torch.ones_like(ids, dtype=torch.float32))
    static = [inputs(*s) for s in sizes]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            work(*s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(*s))
        graphs.append(graph)
    for _ in range(4):
        for i in (0, 1):
            for t, v in zip(static[i], inputs(*sizes[i])):
                t.copy_(v)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], work(*static[i])))


@gpu
def test_a_graph_of_forward_and_backward_replays_the_eager_gradients():
    """Leaves made inside the captured run: no eager graph of theirs lives beside it."""
    import torch
    from qinco_amd import group_rows
    g = torch.Generator("cuda").manual_seed(17)
    n, k, D, E = 700, 3, 40, 90

    def inputs():
        return (torch.randint(-1, E, (n, k), generator=g, device="cuda"), torch.randn(n, D, generator=g, device="cuda"),
                torch.rand(n, k, generator=g, device="cuda"), torch.randn(n, D, generator=g, device="cuda"))

    def work(ids, x, w, d):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        gr = group_rows(ids, E, check=False)
        out = gr.combine(gr.gather(x) * 2.0, w)
        return (out.detach(), *torch.autograd.grad(out, (x, w), d))
    static = inputs()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            work(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(*static)
    for _ in range(4):
        for t, v in zip(static, inputs()):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, work(*static)))


@gpu
def test_together_with_the_search_and_the_look_up_decoder():
    """Codes drawn step by step from a prior's logits, decoded by the look-up decoder, the reconstructions sent to their two nearest lists
    (k-nearest-list search), scaled there and brought back with weights."""
    import torch
    from qinco_amd import group_rows, sample_codes
    from qinco_amd.lut import LutDecoder
    from qinco_amd.search import KnnSearcher
    g = torch.Generator("cuda").manual_seed(9)
    n, M, K, D, E = 700, 4, 256, 32, 100
    u = torch.rand(M, n, generator=g, device="cuda")
    logits = torch.randn(M, n, K, generator=g, device="cuda") * 2
    codes = torch.stack([sample_codes(logits[s], u[s], top_p=0.9) for s in range(M)], 1)
    tables = torch.randn(M, K, D, generator=g, device="cuda")
    dec = LutDecoder(tables.cpu().numpy(), a=np.arange(M))
    x = dec(codes)
    want = sum(to64(tables)[s][codes[:, s].cpu().numpy()] for s in range(M))
    assert np.abs(to64(x) - want).max() <= M * 2.0 ** -24 * np.abs(to64(tables)).max() * M
    centroids = torch.randn(E, D, generator=g, device="cuda")
    knn = KnnSearcher(D)
    ids, dist = knn.search(centroids, x, k=2, return_dist=True)
    gr = check_group(ids, E)
    scale = torch.rand(E, generator=g, device="cuda") + 0.5
    w = torch.softmax(-dist, 1)
    rows = gr.gather(x)
    of_list = torch.repeat_interleave(torch.arange(E, device="cuda"), gr.counts().long())
    out = gr.combine(rows * scale[of_list][:, None], w)
    factor = (to64(w) * to64(scale)[ids.cpu().numpy()]).sum(1)
    assert np.abs(to64(out) - factor[:, None] * to64(x)).max() <= 8 * 2.0 ** -24 * np.abs(factor[:, None] * to64(x)).max()
    first = check_group(codes[:, 0], K)                                              # an index's rows by their first code
    moved = first.gather(codes.to(torch.uint8))
    assert bool((moved[:, 0].diff().int() >= 0).all())
    knn.close(), dec.close()


# ------------------------------------------------------------------------------------------------ far tails, long rows, many rows
def tail_border(V, e, x):
    """One code of mass 1 at index 0, V - 1 of mass e behind it (exact, a Fraction): the code that a share x of the total falls on."""
    at = (x * (1 + (V - 1) * e) - 1) / e                      # tail masses behind the peak's
    return 0 if at < 0 else 1 + int(at)


@gpu
@pytest.mark.parametrize("V,gap", [(60, 33.0), (100, 34.0), (200, 35.0), (500, 35.0), (600, 37.0), (1500, 36.5), (4099, 35.0), (10240, 35.0), (20480, 33.5), (20480, 27.0), (20481, 33.5), (70001, 32.0), (1 << 20, 30.0),
                                   ((1 << 22) + 1, 27.0), (1 << 24, 28.0), (1 << 24, 27.0)])
def test_sample_flat_tails_far_below_the_largest_logit(V, gap):
    """A tail whose codes have 2^-39 to 2^-54 of the largest one's mass each is drawn as often as its share of the row says.  Against whole
    fractions.  A code's mass is held to 2^-44 of itself (the exponential) and a step of at most 2.25 2^-61 of the row's total (up to 512 codes of
    2^-62 for each power of two in V), products with u and p to 2^-52: the code drawn is that many tail masses off at most."""
    import torch
    from fractions import Fraction as Fr
    from decimal import Decimal, localcontext
    from qinco_amd import sample_codes
    with localcontext() as ctx:
        ctx.prec = 60
        e = Fr(Decimal(-gap).exp())
    total, tail = 1 + (V - 1) * e, (V - 1) * e
    step = Fr(9, 1 << 63) if V > 512 else Fr(1, 1 << (62 - (V - 1).bit_length()))
    off = math.ceil((V * step + Fr(1, 1 << 51)) * total / e + V * Fr(1, 1 << 44) + 1)
    assert off < V / 5                                        # (else the case says little)
    z = torch.full((1, V), -gap, device="cuda")
    z[0, 0] = 0.0
    u = [0.3, 1.0 - float(tail / 2), 1.0 - float(tail / 5), 1.0 - float(tail * 4 / 5), 1.0 - float(tail * 2)]
    for n in (5, 300, 2500) if V <= 20480 else (5,):          # (many rows go another way)
        uu = torch.tensor(u, dtype=torch.float64, device="cuda").repeat(n // 5)
        zz = z.expand(n, V)
        for s in (dict(), dict(min_p=1e-30), dict(top_k=V - 1)):
            count = V - (1 if "top_k" in s else 0)            # top-k drops the last of the equal ones
            codes, logp = sample_codes(zz, uu, return_logp=True, **s)
            want = [tail_border(count, e, Fr(x)) for x in u]
            assert want[0] == want[4] == 0 and all(V // 8 < w < V for w in want[1:4])
            codes, logp = codes.view(-1, 5), logp.view(-1, 5)
            assert bool((codes == codes[:1]).all()) and bool((logp == logp[:1]).all())
            got = codes[0].tolist()
            assert got[0] == got[4] == 0 and all(abs(g - w) <= off for g, w in zip(got, want)), (s, got, want, off)
            share = math.log1p(float((count - 1) * e))
            assert abs(float(logp[0, 0]) + share) <= 2.0 ** -24 * share + 2.0 ** -44 + V * float(step)
            assert abs(float(logp[0, 1]) + gap + share) <= 2.0 ** -23 * gap
        keep = 1.0 - float(tail / 2)                          # top-p cuts the tail in the middle
        got = sample_codes(zz, torch.full((n,), 1.0 - 2.0 ** -53, dtype=torch.float64, device="cuda"), top_p=keep)
        assert bool((got == got[0]).all()) and abs(int(got[0]) - tail_border(V, e, Fr(keep))) <= 2 * off


@gpu
@pytest.mark.parametrize("V,dtype", [((1 << 22) + 1, "float32"), (1 << 24, "bfloat16")])
def test_sample_longest_rows(V, dtype):
    """Against the plain statement, whose own sums in 64 bits are good to V 2^-53 of the total."""
    import torch
    from qinco_amd import sample_codes
    g = torch.Generator("cuda").manual_seed(V)
    z = (torch.randn(2, V, generator=g, device="cuda") * 2.5).to(getattr(torch, dtype))
    z[1, : V // 3] = -float("inf")
    z[1, V // 2] = float("nan")
    check_sample(z, torch.rand(2, generator=g, device="cuda"))
    check_sample(z, torch.rand(2, generator=g, device="cuda"), T=0.7, k=1000, p=0.9, m=1e-3)
    z[0, V - 1] = 100.0
    z[1, V - 2:] = 100.0
    assert sample_codes(z, torch.rand(2, generator=g, device="cuda"), temperature=0.0).tolist() == [V - 1, V - 2]


@gpu
@pytest.mark.parametrize("V", [60, 200, 500, 3000, 20000, 70001, 1 << 20])
def test_sample_top_k_among_codes_without_mass(V):
    """Where the k-th code is too far below the largest to have any mass, top-k changes nothing, and costs a long row nothing either: it is not
    sought among the many codes that share its bin."""
    import torch
    from qinco_amd import sample_codes
    g = torch.Generator("cuda").manual_seed(V)
    z = torch.randn(3, V, generator=g, device="cuda") * 2.5
    z[1, V // 3] = 100.0                                                       # one code far above the rest, all different
    z[2] = (z[2] * 4).round()
    u = torch.rand(3, generator=g, device="cuda", dtype=torch.float64)
    for T in (0.02, 0.3):
        for k in (2, 40, V // 3, V - 1):
            check_sample(z, u, T=T, k=k)
            check_sample(z, u, T=T, k=k, p=0.7)
    if V <= 20480:
        return

    def least(**s):
        times = []
        for _ in range(10):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            sample_codes(z[1:2], u[1:2], **s)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)
    assert least(top_k=V // 2) < 4 * least(min_p=1e-30)


# ------------------------------------------------------------------------------------------------ derivatives and traces (no GPU: without the calls)
@pytest.fixture
def no_calls(monkeypatch):
    """Host tensors go through the Python side; the library calls are left out."""
    from qinco_amd import lists, sample
    for m in (lists, sample):
        monkeypatch.setattr(m, "on_device", lambda t, what: t)
        monkeypatch.setattr(m, "on_its_device", lambda index, call, *args: None)
    return lists


def host_groups(lists, n=4, k=2):
    import torch
    place = torch.arange(n * k, dtype=torch.int32)
    return lists.RowGroups(place, place.view(n, k), torch.tensor([0, n * k], dtype=torch.int32))


def test_forward_mode_derivatives_are_refused(no_calls):
    import torch
    import torch.autograd.forward_ad as fa
    g = host_groups(no_calls)
    x, y, w = torch.randn(4, 3), torch.randn(8, 3), torch.rand(4, 2)
    with fa.dual_level():
        dual = lambda t: fa.make_dual(t, torch.ones_like(t))                   # noqa: E731
        for call in (lambda: g.gather(dual(x)), lambda: g.gather(dual(x.cfloat())), lambda: g.combine(dual(y)), lambda: g.combine(dual(y), w), lambda: g.combine(y, dual(w)),
                     lambda: g.combine(dual(y.T.contiguous().T), w)):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError):
                    call()
        assert g.gather(x).shape == (8, 3) and g.gather(x.int()).shape == (8, 3) and g.combine(y, w).shape == (4, 3)   # nothing to lose
        for out, leaves in ((g.gather(x.requires_grad_()), x), (g.combine(y.requires_grad_()), y), (g.combine(y, w.requires_grad_()), (y, w))):
            torch.autograd.grad(out, leaves, torch.ones_like(out), retain_graph=True)
            with pytest.raises(NotImplementedError):                           # ... of a backward pass
                torch.autograd.grad(out, leaves, dual(torch.ones_like(out)))


def test_traces_hold_the_calls_or_are_refused(no_calls):
    """A trace of what torch itself records would answer uninitialised memory."""
    import torch
    from qinco_amd import sample
    g = host_groups(no_calls)
    x, y, w = torch.randn(4, 3), torch.randn(8, 3), torch.rand(4, 2)

    def trace(f, *args):
        return torch.jit.trace(f, args, check_trace=False)
    for f, args, name in ((g.gather, (x,), "_Gather"), (g.gather, (x.to(torch.uint8),), "_Gather"), (g.combine, (y,), "_Combine"), (g.combine, (y, w), "_Combine")):
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                t = trace(lambda *a: f(*a), *args)
            assert "^" + name in str(t.graph) and t(*args).shape == f(*args).shape
    with pytest.raises(RuntimeError, match="cannot be traced"):
        trace(lambda a: no_calls.group_rows(a, 4).order, torch.zeros(5, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        trace(lambda a: sample.sample_codes(a, torch.rand(4)), x)


def test_recording_by_fx_is_refused(no_calls):
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx
    from qinco_amd import sample
    g = host_groups(no_calls)
    x, w = torch.randn(4, 3), torch.rand(4, 2)
    for leaf in (x, x.clone().requires_grad_()):
        for f in (g.gather, lambda a: g.combine(a.repeat(2, 1)), lambda a: g.combine(a.repeat(2, 1), w), lambda a: sample.sample_codes(a, torch.rand(4)),
                  lambda a: no_calls.group_rows((a > 0).to(torch.int64), 4).order):
            f(leaf)
            with pytest.raises(RuntimeError, match="torch.fx"):
                make_fx(lambda a: f(a))(leaf)


@gpu
def test_traced_gather_and_combine_answer_what_they_answer():
    import torch
    g = torch.Generator("cuda").manual_seed(31)
    gr = make_groups(g, 40, 3, 9, True)
    x, y, w = torch.randn(40, 12, generator=g, device="cuda"), torch.randn(120, 12, generator=g, device="cuda"), torch.rand(40, 3, generator=g, device="cuda")
    run = lambda a, b, c: (gr.gather(a) * 2, gr.gather(a.to(torch.uint8)), gr.combine(b), gr.combine(b, c))      # noqa: E731
    traced = torch.jit.trace(run, (x.abs(), y, w))
    for _ in range(3):
        x, y, w = x.roll(1, 0).abs(), y.roll(1, 0), w.roll(1, 0)
        assert all(torch.equal(a, b) for a, b in zip(traced(x, y, w), run(x, y, w)))


def test_log_probabilities_carry_no_derivative(no_calls):
    """As the docstring says, in both modes; the codes neither."""
    import torch
    import torch.autograd.forward_ad as fa
    from qinco_amd.sample import sample_codes
    z, u = torch.randn(4, 8), torch.rand(4)
    codes, logp = sample_codes(z.requires_grad_(), u, temperature=torch.ones(4, requires_grad=True), return_logp=True)
    assert not logp.requires_grad and not codes.requires_grad
    with fa.dual_level():
        assert fa.unpack_dual(sample_codes(fa.make_dual(z.detach(), torch.ones(4, 8)), u, return_logp=True)[1]).tangent is None
    assert "no derivative" in sample_codes.__doc__


@gpu
@pytest.mark.parametrize("V", [50, 200, 500, 3000, 30000])
def test_sample_settings_per_row_that_are_no_settings(V):
    """NaN, infinities and a min_p above 1 in the arrays: what the docstring says they are."""
    import torch
    from qinco_amd import sample_codes
    g = torch.Generator("cuda").manual_seed(V)
    z = torch.randn(12, V, generator=g, device="cuda")
    u = torch.rand(12, generator=g, device="cuda")
    nan, inf = math.nan, math.inf
    row = lambda v, dt=torch.float32: torch.tensor(v, dtype=dt, device="cuda")                                   # noqa: E731
    odd = dict(temperature=row([nan, -inf, -0.0, 1.0] + [0.5] * 8), top_p=row([0.5] * 4 + [nan, inf, -inf, -1.0] + [1.0] * 4),
               min_p=row([0.01] * 8 + [nan, -inf, inf, 7.0]), top_k=row([V + 1, -(1 << 31), (1 << 31) - 1, 0] * 3, torch.int32))
    same = dict(temperature=row([0.0, 0.0, 0.0, 1.0] + [0.5] * 8), top_p=row([0.5] * 4 + [1.0, 1.0, 0.0, 0.0] + [1.0] * 4),
                min_p=row([0.01] * 8 + [0.0, 0.0, 1.0, 1.0]), top_k=row([0] * 12, torch.int32))
    a, b = sample_codes(z, u, return_logp=True, **odd), sample_codes(z, u, return_logp=True, **same)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    first = z.argmax(1)                                       # (all different)
    assert torch.equal(a[0][[0, 1, 2, 6, 7, 10, 11]], first[[0, 1, 2, 6, 7, 10, 11]])
    z[:, ::3] = -inf
    hot = sample_codes(z, u, temperature=torch.full((12,), inf, device="cuda"))        # every finite logit as likely
    assert torch.equal(hot, sample_codes(torch.where(z > -inf, 0.0, z), u))


@gpu
@pytest.mark.parametrize("n,V,dtype", [(2900, 20481, "float16"), (90, 1 << 20, "float32")])
def test_sample_more_long_rows_than_one_batch_holds(n, V, dtype):
    """The workspace holds some 1300 rows of 20481 codes, some 70 of 2^20: what is drawn does not depend on where a batch ends."""
    import torch
    from qinco_amd import sample_codes
    g = torch.Generator("cuda").manual_seed(n)
    z = (torch.randn(n, V, generator=g, device="cuda") * 2.5).to(getattr(torch, dtype))
    z[n // 2] = -float("inf")
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    T = torch.rand(n, generator=g, device="cuda") + 0.2
    T[::7] = 0.0
    for s in (dict(), dict(top_k=40, top_p=0.9, min_p=0.01)):
        codes, logp = sample_codes(z, u, temperature=T, return_logp=True, **s)
        for a in range(0, n, 60):                                              # every row in a batch of its own neighbourhood
            b = min(a + 60, n)
            c, l = sample_codes(z[a:b], u[a:b], temperature=T[a:b], return_logp=True, **s)
            assert torch.equal(c, codes[a:b]) and torch.equal(l, logp[a:b])
        assert int(codes[n // 2]) == -1 and torch.equal(z[::7].gather(1, codes[::7, None])[:, 0], z[::7].amax(1))
    rows = [0, 1, n // 2, n - 2, n - 1]
    check_sample(z[rows], u[rows].contiguous(), T=T[rows].cpu().numpy(), k=40, p=0.9, m=0.01)


@gpu
@pytest.mark.parametrize("V", [60, 200, 500, 3000, 30000])
def test_sample_rows_behind_four_giga_elements(V):
    """Rows 2^23 elements apart: the last ones begin behind 2^32 elements."""
    import torch
    from qinco_amd import sample_codes
    g = torch.Generator("cuda").manual_seed(V)
    n, stride = 520, 1 << 23
    store = torch.empty((n - 1) * stride + V, dtype=torch.bfloat16, device="cuda")
    z = store.as_strided((n, V), (stride, 1))
    near = (torch.randn(n, V, generator=g, device="cuda") * 2.5).bfloat16()
    z.copy_(near)
    u = torch.rand(n, generator=g, device="cuda")
    for s in (dict(), dict(top_k=30, top_p=0.9)):
        assert torch.equal(sample_codes(z, u, **s), sample_codes(near, u, **s))


@gpu
def test_gather_and_combine_behind_two_to_the_32_elements():
    """More than 2^32 elements of one byte (rows of an odd number of bytes: moved byte by byte) and of two, in both directions."""
    import torch
    from qinco_amd import group_rows
    n, k, D = 2_200_000, 2, 1001
    assert n * k * D > 1 << 32
    r = torch.arange(n, device="cuda")
    gr = group_rows(torch.stack([r, r], 1), n)                                  # row r in places 2 r, 2 r + 1
    x = torch.randint(0, 256, (n, D), device="cuda", dtype=torch.uint8)
    out = gr.gather(x)
    assert torch.equal(out[::2], x) and torch.equal(out[1::2], x)
    del x
    y = out.to(torch.bfloat16)
    del out
    w = torch.tensor([[1.0, -0.5]], device="cuda").expand(n, 2).contiguous()
    got = gr.combine(y, w)
    assert torch.equal(got, y[::2] * 0.5)
    dy, dw = gr._combine_grad(got, y, w, True, True)
    assert torch.equal(dy[::2], got) and torch.equal(dy[1::2], got * -0.5)
    for i in (0, n // 2, n - 1):
        want = float((got[i].double() * y[2 * i].double()).sum())
        assert abs(float(dw[i, 0]) - want) <= D * 2.0 ** -24 * want and float(dw[i, 0]) == float(dw[i, 1])


@gpu
@pytest.mark.parametrize("V,n", [(60, 64), (60, 4096), (120, 64), (120, 4096), (250, 64), (250, 4096), (500, 64), (1000, 64), (1000, 512), (2048, 64), (2048, 512), (4099, 64), (4099, 512),
                                 (10000, 64), (10000, 512), (20480, 64), (70001, 64), (1 << 20, 64), (1 << 22, 64)])
def test_sample_draws_and_cuts_within_the_stated_distance_of_a_border(V, n):
    """u, and top_p, next to the borders between codes, as far from them as the stated bound, against sums of 64-bit mantissas."""
    import torch
    from qinco_amd import sample_codes
    rs = np.random.RandomState(V)
    near = 2.0 ** -52 + 2.0 ** -44 + (V * 2.0 ** -53 if V <= 512 else 2.25 * V * 2.0 ** -61)
    for T, spread in ((1.0, 2.5), (0.37, 4.0), (3.0, 0.5)):
        z = (rs.randn(V) * spread).astype(np.float32)
        top = np.longdouble(z.max())
        e = np.exp((z.astype(np.longdouble) - top) / np.longdouble(T))
        heavy = np.flatnonzero(e / e.sum() > 16 * near)
        dev = torch.from_numpy(z).cuda().expand(n, V)
        # draws: above and below the border behind code i
        run = np.cumsum(e) / e.sum()
        i = rs.choice(heavy[:-1], n // 2)
        u = np.concatenate([run[i] - near, run[i] + near]).astype(np.float64)
        for s in (dict(), dict(min_p=1e-30)):
            got = sample_codes(dev, torch.from_numpy(u).cuda(), temperature=T, **s).cpu().numpy()
            assert np.all((run[got] + near > u) & (run[got] - e[got] / e.sum() - near <= u))
            assert np.array_equal(got[: n // 2], i)                                    # (heavy codes: just before their end)
        # top-p: the codes kept are the first r by logit; u = 0 draws the lowest kept index, u -> 1 the highest
        order = np.argsort(-z, kind="stable")
        before = np.cumsum(e[order]) / e.sum()
        for r in rs.choice(np.flatnonzero(e[order] / e.sum() > 16 * near)[:-1], 8):
            for p, kept in ((before[r] - near, r + 1), (before[r] + near, r + 2)):
                if not 0 < p < 1:
                    continue
                ends = torch.tensor([0.0, 1.0 - 2.0 ** -53], dtype=torch.float64, device="cuda").repeat(n // 2)
                got = sample_codes(dev, ends, temperature=T, top_p=float(p)).cpu().numpy()
                share = e[np.sort(order[:kept])] / e[order[:kept]].sum()
                if share[-1] > near:
                    assert np.all(got[0::2] == order[:kept].min()) and np.all(got[1::2] == order[:kept].max()), (T, r, p)


def test_workspaces_at_odd_addresses_are_refused(lib):
    """Decided on the host, before anything is launched: their 64-bit words and atomics would not be aligned."""
    from qinco_amd import _lib
    P = _lib.QincoSampleParams
    params = P(struct_bytes=C.sizeof(P), temperature=1.0, top_p=0.5)
    buf = (C.c_char * 64)()
    at = (C.addressof(buf) + 15) // 16 * 16
    for off in (1, 2, 4, 8):
        assert lib.qinco_sample_codes(at, 0, 30000, 2, 30000, at, 0, C.byref(params), at, 0, None, at + off, 1 << 40, None) == -1
        assert b"qinco_sample_codes" in lib.qinco_last_error() and b"aligned" in lib.qinco_last_error()
        assert lib.qinco_group_rows(at, 0, 1, 4, 1, 8, at, at, at, None, at + off, 1 << 40, None) == -1
        assert b"qinco_group_rows" in lib.qinco_last_error() and b"aligned" in lib.qinco_last_error()


@pytest.mark.parametrize("needs_grad", [False, True])
def test_traces_look_at_the_tensors_they_get(no_calls, monkeypatch, needs_grad):
    """What was looked at while tracing says nothing of the tensors that a trace gets later: other rows, types and strides."""
    import torch
    seen = []
    monkeypatch.setattr(no_calls, "on_its_device", lambda index, call, *args: seen.append(args))
    g = host_groups(no_calls)
    x, y, w = torch.randn(4, 3), torch.randn(8, 3), torch.rand(4, 2)
    gather = torch.jit.trace(lambda a: g.gather(a), (x.requires_grad_(needs_grad),), check_trace=False)
    combine = torch.jit.trace(lambda a, b: g.combine(a, b), (y.requires_grad_(needs_grad), w), check_trace=False)
    for bad in (x[:3], x[0], torch.randn(5, 3)):
        with pytest.raises(Exception, match="x must be"):
            gather(bad)
    for a, b in ((y[:7], w), (y, w[:3]), (y, w.double()), (y.double(), w), (y, torch.rand(2, 4))):
        with pytest.raises(Exception, match="must be"):
            combine(a, b)
    seen.clear()
    wide = torch.randn(9, 4)
    assert gather(wide.T).shape == (8, 9) and seen[0][1] == 9 * 4                       # rows of 9 elements next to each other
    seen.clear()
    combine(torch.randn(9, 8).T, torch.rand(2, 4).T)
    assert seen[0][2:4] == (9, 9)


@gpu
def test_traces_with_other_rows_than_they_were_made_with():
    import torch
    g = torch.Generator("cuda").manual_seed(33)
    gr = make_groups(g, 40, 3, 9, True)
    x, y, w = torch.randn(40, 12, generator=g, device="cuda"), torch.randn(120, 12, generator=g, device="cuda"), torch.rand(40, 3, generator=g, device="cuda")
    run = lambda a, b, c: (gr.gather(a), gr.combine(b, c))                                        # noqa: E731
    traced = torch.jit.trace(run, (x, y, w))
    for D in (1, 7, 130):
        a, b = torch.randn(D, 40, generator=g, device="cuda").T, torch.randn(D, 120, generator=g, device="cuda").T.bfloat16()
        got, want = traced(a, b, w.T.contiguous().T), run(a, b, w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(Exception, match="x must be"):
        traced(x[:39], y, w)


@gpu
@pytest.mark.parametrize("V", [200, 500, 3000, 30000, 300000])
def test_sample_logits_over_the_whole_range_at_huge_temperatures(V):
    """Differences that fp32 does not hold, at temperatures that bring them back to size 1."""
    import torch
    g = torch.Generator("cuda").manual_seed(V)
    z = torch.full((5, V), -3.0e38, device="cuda")
    z[0, V // 2] = 3.0e38
    z[1] = (torch.rand(V, generator=g, device="cuda") * 2 - 1) * 3.4e38
    z[2, ::2] = 3.0e38
    z[3, : V // 2] = -float("inf")
    z[3, V - 1] = 3.4e38
    z[4, V // 3] = float("inf")
    for T in (1e38, 3e38, 1e39, 1e42, 1e45, 1e300):
        for s in (dict(), dict(p=0.7), dict(k=V // 3, p=0.9, m=0.3)):
            check_sample(z, torch.rand(5, generator=g, device="cuda", dtype=torch.float64), T=T, **s)
