"""Cases of the operators between a model that answers in codes and the codec: sampling codes from logits, grouping rows by inverted
list, carrying rows to their groups and back with weights, and the gradients of both.

`run` computes them with elementary torch operations in 64 or 32 bits, or, where `own` is true, through qinco_amd."""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16, "uint8": torch.uint8, "int32": torch.int32,
          "int64": torch.int64}


def listed():
    return [
        # the next code of one sequence: a codebook of 256, the smallest call
        {"name": "sample one row", "op": "sample", "n": 1, "V": 256, "dtype": "float32", "temperature": 1.0, "top_k": 0, "top_p": 0.95,
         "min_p": 0.0, "mask": 0.0, "per_row": False},
        # a decode batch of the search, every row with its own settings
        {"name": "sample a batch", "op": "sample", "n": 12288, "V": 256, "dtype": "bfloat16", "temperature": 0.8, "top_k": 50, "top_p": 0.95,
         "min_p": 0.02, "mask": 0.0, "per_row": True},
        # a codebook of odd size, a quarter of it ruled out by a prefix constraint, top-k alone
        {"name": "sample masked", "op": "sample", "n": 1000, "V": 4099, "dtype": "float16", "temperature": 1.0, "top_k": 40, "top_p": 1.0,
         "min_p": 0.0, "mask": 0.25, "per_row": False},
        # one inverted list of 2^20 for each of a few queries
        {"name": "sample a list", "op": "sample", "n": 16, "V": 1 << 20, "dtype": "float32", "temperature": 0.7, "top_k": 0, "top_p": 0.9,
         "min_p": 0.0, "mask": 0.0, "per_row": False},
        # a few vectors by their first code
        {"name": "group a few", "op": "group", "n": 50, "k": 1, "E": 256, "dtype": "uint8", "drop": 0.0, "skew": False},
        # queries by their probed lists, some probes void
        {"name": "group probes", "op": "group", "n": 12289, "k": 8, "E": 1024, "dtype": "int64", "drop": 0.1, "skew": True},
        # filling an index: a million vectors by inverted list
        {"name": "group an index", "op": "group", "n": 1 << 20, "k": 1, "E": 1 << 20, "dtype": "int32", "drop": 0.0, "skew": False},
        # the code rows of that index moved into list order
        {"name": "gather codes", "op": "gather", "n": 1000000, "k": 1, "D": 8, "E": 1 << 16, "dtype": "uint8", "drop": 0.0, "grad": False},
        # a training batch carried to its lists, forward and backward
        {"name": "gather and gradient", "op": "gather", "n": 65536, "k": 4, "D": 128, "E": 1024, "dtype": "bfloat16", "drop": 0.0, "grad": True},
        # a few queries back from their probes
        {"name": "combine a few", "op": "combine", "n": 37, "k": 8, "D": 128, "E": 256, "dtype": "float32", "drop": 0.0, "grad": False},
        # the training batch back with weights, forward and backward
        {"name": "combine and gradient", "op": "combine", "n": 65536, "k": 8, "D": 128, "E": 1024, "dtype": "bfloat16", "drop": 0.0, "grad": True},
        # rows of an odd width, some probes void
        {"name": "combine odd rows", "op": "combine", "n": 30011, "k": 5, "D": 101, "E": 999, "dtype": "float32", "drop": 0.1, "grad": True},
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of its range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "group", "gather", "combine"])
    if op == "sample":
        V = 256 if rng.random() < 0.3 else _spread(rng, 2, 1 << 20)
        n = _spread(rng, 1, max(1, min(65536, (1 << 24) // V)))
        return {"op": op, "n": n, "V": V, "dtype": rng.choice(["float32", "float16", "bfloat16"]),
                "temperature": round(rng.uniform(0.3, 2.0), 2), "top_k": rng.choice([0, 1, _spread(rng, 1, V)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.05, 0.99), 2)]), "min_p": rng.choice([0.0, round(rng.uniform(0.001, 0.2), 3)]),
                "mask": rng.choice([0.0, 0.5]), "per_row": rng.random() < 0.5}
    k = rng.choice([1, 1, 2, 3, 4, 8, 16])
    E = _spread(rng, 1, 1 << 20)
    drop = rng.choice([0.0, 0.1])
    if op == "group":
        n = _spread(rng, 1, (1 << 20) // k)
        dtype = rng.choice(["int64", "int32"] + (["uint8"] if E <= 256 else []))
        return {"op": op, "n": n, "k": k, "E": E, "dtype": dtype, "drop": 0.0 if dtype == "uint8" else drop, "skew": rng.random() < 0.5}
    D = rng.choice([8, 32, 96, 100, 128, 200, 256, 384, 768, _spread(rng, 1, 1024)])
    n = _spread(rng, 1, max(1, min(1 << 20, (1 << 25) // (k * D))))
    dtype = rng.choice(["float32", "float16", "bfloat16"] + (["uint8", "int32", "int64"] if op == "gather" else []))
    return {"op": op, "n": n, "k": k, "D": D, "E": E, "dtype": dtype, "drop": drop, "grad": "int" not in dtype and rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------- inputs
def _lists(case, g, dev):
    """Lists of every row: uniform or with a long tail; a share of them -1 (no list)."""
    n, k, E = case["n"], case["k"], case["E"]
    r = torch.rand(n, k, generator=g, device=dev, dtype=torch.float64)
    ids = (r ** 3 if case.get("skew") else r).mul(E).long().clamp_(0, E - 1)
    if case["drop"] > 0:
        ids[torch.rand(n, k, generator=g, device=dev) < case["drop"]] = -1
        ids[n // 2] = -1
    return ids


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "sample":
        n, V = case["n"], case["V"]
        x = torch.randn(n, V, generator=g, device=dev) * 2.5
        if case["mask"] > 0:
            x[torch.rand(n, V, generator=g, device=dev) < case["mask"]] = float("-inf")
            x[60::61] = float("-inf")
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["u"] = torch.rand(n, generator=g, device=dev)
        for name in ("temperature", "top_k", "top_p", "min_p"):
            s[name] = case[name]
        if case["per_row"]:
            def around():
                return 0.5 + torch.rand(n, generator=g, device=dev)
            s["temperature"] = case["temperature"] * around()
            s["top_k"] = (case["top_k"] * around()).round().to(torch.int32)
            s["top_p"] = (case["top_p"] * around()).clamp(max=1.0)
            s["min_p"] = case["min_p"] * around()
        return s
    s["lists"] = _lists(case, g, dev)
    if case["op"] == "group":
        s["lists"] = s["lists"].to(DTYPES[case["dtype"]])
        return s
    s["order"], s["place"], s["offsets"] = _plain_group(s.pop("lists"), case["E"])
    n, k, D, dt = case["n"], case["k"], case["D"], DTYPES[case["dtype"]]

    def rows(m):
        if dt.is_floating_point:
            return torch.randn(m, D, generator=g, device=dev).to(dt)
        return torch.randint(0, 256, (m, D), generator=g, device=dev).to(dt)
    if case["op"] == "gather":
        s["x"] = rows(n)
        s["dout"] = rows(n * k) if case["grad"] else None
    else:
        s["y"] = rows(n * k)
        if case["drop"] > 0:  # rows that no entry owns hold whatever was there
            s["y"][s["order"] < 0] = float("nan")
        s["weights"] = torch.softmax(torch.randn(n, k, generator=g, device=dev), 1)
        s["dout"] = rows(n) if case["grad"] else None
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _column(v, like):
    return v.double()[:, None] if torch.is_tensor(v) else torch.full((1, 1), v, dtype=torch.float64, device=like.device)


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    """In 64 bits: a random number next to a border between two codes has to fall on the same side."""
    z = logits.double()
    z = torch.where(z.isnan(), float("-inf"), z)
    n, V = z.shape
    T, k, p, m = (_column(v, z) for v in (temperature, top_k, top_p, min_p))
    top = z.max(1, keepdim=True).values
    usable = z > float("-inf")
    e = torch.where(usable, torch.where(z == top, 1.0, torch.exp((z - top) / T)), 0.0)
    order = torch.sort(z, dim=1, descending=True, stable=True).indices
    es = e.gather(1, order)
    rank = torch.arange(V, device=z.device)[None]
    es = torch.where((rank < k) | (k <= 0), es, 0.0)
    before = torch.cat([torch.zeros_like(es[:, :1]), es.cumsum(1)], 1)
    keep = (es > 0) & ((before[:, :-1] < p * before[:, -1:]) | (p >= 1) | (rank == 0)) & (es >= m)
    keep = torch.zeros_like(usable).scatter(1, order, keep)
    mass = torch.where(keep, e, 0.0).cumsum(1)
    code = (mass <= u.double()[:, None] * mass[:, -1:]).sum(1, keepdim=True).clamp(max=V - 1)
    logp = torch.where(z.gather(1, code) == top, 0.0, (z.gather(1, code) - top) / T) - mass[:, -1:].log()
    greedy = T <= 0
    code, logp = torch.where(greedy, order[:, :1], code), torch.where(greedy, 0.0, logp)
    none = ~usable.any(1, keepdim=True)
    code, logp = torch.where(none, -1, code), torch.where(none, float("-inf"), logp)
    return code[:, 0], logp[:, 0].float()


def _plain_group(lists, E):
    key = lists.reshape(-1).long()
    ok = (key >= 0) & (key < E)
    N = key.numel()
    slot = torch.arange(N, device=key.device)
    key = torch.where(ok, key, E)
    order = torch.sort(key, stable=True).indices
    counts = torch.zeros(E + 1, dtype=torch.int64, device=key.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = counts.cumsum(0) - counts
    place = torch.empty_like(order).scatter_(0, order, slot)
    order = torch.where(slot < offsets[E], order, -1)
    place = torch.where(ok, place, -1).reshape(lists.shape[0], -1)
    return order.int(), place.int(), offsets.int()


def _plain_gather(x, order, place, dout):
    k = place.shape[1]
    used = (order >= 0)[:, None]
    out = torch.where(used, x[order.clamp(min=0) // k], torch.zeros((), dtype=x.dtype, device=x.device))
    if dout is None:
        return out
    dx = torch.where((place >= 0)[:, :, None], dout.float()[place.clamp(min=0)], 0.0).sum(1)
    return out, dx.to(x.dtype)


def _plain_combine(y, weights, order, place, dout):
    n, k = place.shape
    w = weights.float()
    yk = torch.where((place >= 0)[:, :, None], y.float()[place.clamp(min=0)], 0.0)
    out = (w[:, :, None] * yk).sum(1).to(y.dtype)
    if dout is None:
        return out
    entry = order.clamp(min=0)
    dy = torch.where((order >= 0)[:, None], w.reshape(-1)[entry][:, None] * dout.float()[entry // k], 0.0).to(y.dtype)
    dw = (dout.float()[:, None, :] * yk).sum(2)
    return out, dy, dw


# ---------------------------------------------------------------------------------------------- one pass
def _own(s):
    from qinco_amd.lists import RowGroups, group_rows
    from qinco_amd.sample import sample_codes
    case = s["case"]
    if case["op"] == "sample":
        return sample_codes(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                            return_logp=True)
    if case["op"] == "group":
        g = group_rows(s["lists"], case["E"], check=False)
        return g.order, g.place, g.offsets
    g = RowGroups(s["order"], s["place"], s["offsets"])
    if case["op"] == "gather":
        if s["dout"] is None:
            return g.gather(s["x"])
        x = s["x"].detach().requires_grad_()
        out = g.gather(x)
        return out.detach(), torch.autograd.grad(out, x, s["dout"])[0]
    if s["dout"] is None:
        return g.combine(s["y"], s["weights"])
    y, w = s["y"].detach().requires_grad_(), s["weights"].detach().requires_grad_()
    out = g.combine(y, w)
    return (out.detach(), *torch.autograd.grad(out, (y, w), s["dout"]))


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "sample":
        return _plain_sample(*(state[name] for name in ("logits", "u", "temperature", "top_k", "top_p", "min_p")))
    if op == "group":
        return _plain_group(state["lists"], state["case"]["E"])
    if op == "gather":
        return _plain_gather(state["x"], state["order"], state["place"], state["dout"])
    return _plain_combine(state["y"], state["weights"], state["order"], state["place"], state["dout"])


def work(case):
    size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    n = case["n"]
    if case["op"] == "sample":
        return {"bytes": n * (case["V"] * size + 4 + 12), "flops": 2 * n * case["V"]}
    N = n * case["k"]
    if case["op"] == "group":
        return {"bytes": N * (size + 8) + 4 * (case["E"] + 1), "flops": 0}
    row = case["D"] * size
    if case["op"] == "gather":
        once = n * row + N * (row + 4)
        return {"bytes": once * (2 if case["grad"] else 1), "flops": N * case["D"] if case["grad"] else 0}
    forward = N * (row + 8) + n * row
    backward = N * (2 * row + 12) + n * row
    return {"bytes": forward + (backward if case["grad"] else 0), "flops": N * case["D"] * (5 if case["grad"] else 2)}


# ---------------------------------------------------------------------------------------------- by definition, in 64 bits
def _exact_sample(s):
    """Row by row as it is written down: sort, cut, renormalise, walk the kept codes in index order."""
    z = s["logits"].double().cpu().numpy()
    n, V = z.shape
    u = s["u"].double().cpu().numpy()
    T, k, p, m = (np.broadcast_to(v.double().cpu().numpy() if torch.is_tensor(v) else np.float64(v), (n,))
                  for v in (s["temperature"], s["top_k"], s["top_p"], s["min_p"]))
    codes, logps = np.full(n, -1, np.int64), np.full(n, -np.inf)
    for r in range(n):
        at = np.flatnonzero(z[r] > -np.inf)
        if not len(at):
            continue
        at = at[np.argsort(-z[r][at], kind="stable")]
        if k[r] > 0:
            at = at[: int(k[r])]
        e = np.exp((z[r][at] - z[r][at[0]]) / T[r])
        if p[r] < 1:
            mass = np.cumsum(e)
            last = 1 + int(np.searchsorted(mass, p[r] * mass[-1], side="left"))
            at, e = at[:last], e[:last]
        at, e = at[e >= m[r]], e[e >= m[r]]
        back = np.argsort(at)
        at, e = at[back], e[back]
        mass = np.cumsum(e)
        i = min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), len(at) - 1)
        codes[r], logps[r] = at[i], np.log(e[i] / mass[-1])
    return codes, logps


def exact(case, seed):
    if case["op"] == "sample" and case["n"] * (case["V"] + 600) > 1 << 25:
        return None
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    if case["op"] == "group":
        ids = s["lists"].cpu().numpy().astype(np.int64).reshape(-1)
        E = case["E"]
        entries = np.flatnonzero((ids >= 0) & (ids < E))
        entries = entries[np.lexsort((entries, ids[entries]))]
        order, place = np.full(ids.size, -1, np.int32), np.full(ids.size, -1, np.int32)
        order[: len(entries)] = entries
        place[entries] = np.arange(len(entries))
        offsets = np.searchsorted(ids[entries], np.arange(E + 1), side="left").astype(np.int32)
        return order, place.reshape(case["n"], case["k"]), offsets
    n, k, D = case["n"], case["k"], case["D"]
    used = torch.nonzero(s["order"] >= 0)[:, 0]
    entry = s["order"][used].long()
    row = entry // k
    new = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device=used.device)  # noqa: E731
    if case["op"] == "gather":
        if not s["x"].is_floating_point():
            out = torch.zeros(n * k, D, dtype=s["x"].dtype, device=used.device)
            out[used] = s["x"][row]
            return out
        out = new(n * k, D)
        out[used] = s["x"].double()[row]
        return out if s["dout"] is None else (out, new(n, D).index_add_(0, row, s["dout"].double()[used]))
    w = s["weights"].double().reshape(-1)[entry]
    yu = s["y"].double()[used]
    out = new(n, D).index_add_(0, row, w[:, None] * yu)
    if s["dout"] is None:
        return out
    du = s["dout"].double()[row]
    dy, dw = new(n * k, D), new(n * k)
    dy[used] = w[:, None] * du
    dw[entry] = (du * yu).sum(1)
    return out, dy, dw.reshape(n, k)
