"""The paged 8-bit key/value cache as timed cases: writing it (quantising tokens as they come), reading it back, and
attention over it -- single tokens, a few tokens, chunks of a prompt.

The cache holds keys and values as INT8 or E4M3 codes in pages of `page` tokens, with one f32 scale for each page and kv
head: k, v [pages, Hkv, page, D], k_scale, v_scale [pages, Hkv].  A sequence owns the pages its row of the page table names;
token t lies in row t % page of page table[t // page].  New tokens of all sequences are packed in one [T, H, D] tensor,
sequence b's in rows starts[b] .. starts[b + 1]; they are the LAST tokens of the sequence: `lengths` counts them in.

Writing gives a page the scale of the largest value it has received: amax / 127 for INT8, the least power of two that is
at least amax / 448 for E4M3, neither below 2^-60.  When later tokens raise the scale of a page, the codes that are there
are rounded again to the new scale.  An optional offset per kv head and channel, `k_mean`, is subtracted from the keys before they are
quantised and added when they are read back; attention does not depend on it, since it moves all logits of a row alike.
Attention is softmax(q k^T / sqrt(D)) v over the values the codes stand for, query heads in groups of Hq / Hkv per kv head;
with `causal` a token sees the keys up to its own position.  A row that sees no key is zero.

`own` false: the plain form, elementary torch operations in 32 bits, sequence by sequence.  `own` true: the package's
kernels.
"""
import torch

own = False

GOLDEN = 0.6180339887498949
FLOOR = 2.0 ** -60


def _case(name, kind, B, Hq, Hkv, D, L, new=1, page=64, fp8=False, dtype="bf16", ragged=False, idle=0, mean=False,
          causal=True):
    return {"name": name, "kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "L": L, "new": new, "page": page, "fp8": fp8,
            "dtype": dtype, "ragged": ragged, "idle": idle, "mean": mean, "causal": causal}


def listed():
    return [
        # one short sequence, one token: written and attended (a step returns what it changed in the cache too); the smallest call, all
        # latency
        _case("step_single", "step", 1, 12, 12, 64, 197, page=16),
        # token generation for a small batch of long conversations, grouped heads
        _case("decode_gqa", "attend", 8, 32, 8, 128, 8192),
        # a server's batch: lengths of all sizes, small pages, a few idle slots (length 0), keys with an offset per channel
        _case("decode_ragged", "step", 64, 32, 8, 128, 4096, page=16, ragged=True, idle=3, mean=True),
        # one very long document, where the work has to be split over the tokens
        _case("decode_long", "attend", 1, 32, 8, 128, 131072, page=128, fp8=True),
        # full-precision queries, one kv head per query head, odd lengths
        _case("decode_f32", "attend", 8, 16, 16, 64, 2047, page=32, dtype="f32", ragged=True),
        # five proposed tokens of each sequence verified at once, sixteen query heads on one kv head
        _case("verify", "step", 16, 32, 2, 128, 3001, new=5, fp8=True, ragged=True),
        # a chunk of a long prompt against what is in the cache
        _case("chunk", "attend", 2, 32, 8, 128, 16384, new=1024, page=128),
        # whole short prompts of different lengths, from an empty cache
        _case("prompts", "step", 4, 16, 16, 64, 789, new=789, page=32, fp8=True, ragged=True),
        # long prompts written to the cache in one call (and the written tokens read back)
        _case("write_prompt", "write", 8, 8, 8, 128, 4096, new=4096, mean=True),
        # one token of each of many sequences written into open pages (and those pages read back)
        _case("write_tokens", "write", 64, 8, 8, 128, 4096, page=16, fp8=True, ragged=True),
        # long contexts read back, for a layer or a machine that wants them in 16 bits
        _case("read_context", "read", 4, 8, 8, 128, 32768, page=128, mean=True),
        # short ragged contexts read back in 32 bits
        _case("read_f32", "read", 3, 2, 2, 64, 3001, page=16, fp8=True, dtype="f32", ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    most = {"bytes": 6e8, "flops": 2.5e11}  # of the listed cases: what the largest of them reads or computes
    while True:
        kind = rng.choice(["attend", "attend", "step", "step", "write", "read"])
        B = _log_int(rng, 1, 64)
        L = _log_int(rng, 1, 131072)
        new = 1
        if kind == "write" or (kind != "read" and rng.random() < 0.5):
            new = min(L, _log_int(rng, 1, 4096))
        Hkv = rng.choice([1, 2, 3, 4, 8, 12, 16])
        Hq = Hkv * rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 16])
        case = _case("", kind, B, Hq, Hkv, rng.choice([64, 128]), L, new, rng.choice([16, 32, 64, 128]), rng.random() < 0.5,
                     "f32" if rng.random() < 0.3 else "bf16", rng.random() < 0.6, rng.choice([0, 0, 1]) if B > 1 else 0,
                     rng.random() < 0.4, rng.random() < 0.85)
        del case["name"]
        w = work(case)
        # the plain form holds the scores of one sequence; it works one sequence after the other
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and Hq * new * L <= 6e8 and B * L <= 2 ** 18:
            return case


def _sequences(case):
    """(length, new tokens) of each sequence, the new ones counted in; idle slots have length 0 and one row."""
    B, L, new = case["B"], case["L"], case["new"]
    seqs = []
    for b in range(B):
        if b >= B - case["idle"]:
            seqs.append((0, 1))
            continue
        at = (b * GOLDEN) % 1.0 if case["ragged"] else 0.0
        length = L - int(at * (L - 1))
        n = max(1, new - int(at * new)) if case["ragged"] and new > 8 else new
        seqs.append((length, min(n, length)))
    return seqs


def _outputs(case):
    """Attention returns its rows; what changes the cache returns the values that the changed pages stand for."""
    return {"attend": ("o",), "step": ("o", "k", "v"), "write": ("k", "v"), "read": ("k", "v")}[case["kind"]]


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _scale_of(amax, fp8):
    if not fp8:
        return torch.clamp_min(amax / 127.0, FLOOR)
    f, e = torch.frexp(amax)  # amax = f * 2^e with f in [1/2, 1); 448 = 0.875 * 2^9
    e = torch.where(f > 0.875, e - 8, e - 9)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e.to(amax.dtype)), torch.zeros_like(amax)).clamp_min(FLOOR)


def _encode(x, scale, fp8):
    """Codes of x [..., D] for a scale that broadcasts over it."""
    y = x * (1.0 / scale)
    if fp8:
        return y.to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.round(y).clamp(-127, 127).to(torch.int8)


def _values(codes):
    return (codes.view(torch.float8_e4m3fn) if codes.dtype == torch.uint8 else codes).float()


def _write(codes, scales, x, pages, first, page, fp8):
    """Tokens x [n, Hkv, D] (f32) become the positions first .. first + n of the sequence that owns `pages`."""
    n, H, D = x.shape
    j0, off = first // page, first % page
    nb = (off + n + page - 1) // page
    own_pages = pages[j0:j0 + nb].long()
    new = torch.zeros(nb * page, H, D, device=x.device)
    new[off:off + n] = x
    new = new.view(nb, page, H, D).transpose(1, 2)
    at = torch.arange(nb * page, device=x.device).view(nb, 1, page, 1)
    amax = new.abs().amax(dim=(2, 3))
    old_scale = scales[own_pages]
    scale = _scale_of(amax, fp8)
    if off:
        scale[0] = torch.maximum(scale[0], old_scale[0])
    spread = scale[:, :, None, None]
    old = codes[own_pages]
    out = torch.where((at >= off) & (at < off + n), _encode(new, spread, fp8), old)
    if off:
        ratio = (old_scale[0] / scale[0])[:, None, None]
        moved = _values(old[0]) * ratio
        moved = moved.to(torch.float8_e4m3fn).view(torch.uint8) if fp8 else torch.round(moved).to(torch.int8)
        out[0, :, :off] = moved[:, :off]
    codes[own_pages] = out
    scales[own_pages] = scale


def _gather(codes, scales, pages, length, page):
    """The first `length` tokens of a sequence, [length, Hkv, D] in f32."""
    at = pages[:(length + page - 1) // page].long()
    x = _values(codes[at]) * scales[at][:, :, None, None]
    return x.transpose(1, 2).reshape(-1, codes.shape[1], codes.shape[3])[:length]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, Hq, Hkv, D, page, fp8 = (case[k] for k in ("B", "Hq", "Hkv", "D", "page", "fp8"))
    dtype, seqs = _dtype(case), _sequences(case)
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
    counts = [(length + page - 1) // page for length, _ in seqs]
    pool = sum(counts) + 3
    order = torch.randperm(pool, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((B, max(max(counts), 1)), -1, dtype=torch.int32, device="cuda")
    code_type = torch.uint8 if fp8 else torch.int8
    state = {"case": case, "seqs": seqs, "table": table,
             "k": torch.zeros(pool, Hkv, page, D, dtype=code_type, device="cuda"),
             "v": torch.zeros(pool, Hkv, page, D, dtype=code_type, device="cuda"),
             "k_scale": torch.zeros(pool, Hkv, device="cuda"), "v_scale": torch.zeros(pool, Hkv, device="cuda")}
    # keys have a large offset in some channels, values none; with `mean` a calibrated offset is known
    offset = 2.0 * rand(Hkv, D) if case["mean"] else torch.zeros(Hkv, D, device="cuda")
    state["k_mean"] = offset + 0.05 * rand(Hkv, D) if case["mean"] else None
    taken = 0
    for b, (length, n) in enumerate(seqs):
        pages = order[taken:taken + counts[b]]
        table[b, :counts[b]] = pages
        taken += counts[b]
        held = length - n if case["kind"] in ("step", "write") else length
        if held > 0:
            k = rand(held, Hkv, D) + offset - (state["k_mean"] if case["mean"] else 0.0)
            _write(state["k"], state["k_scale"], k, pages, 0, page, fp8)
            _write(state["v"], state["v_scale"], rand(held, Hkv, D), pages, 0, page, fp8)
    T = sum(n for _, n in seqs)
    fused = rand(T, (Hq + 2 * Hkv) * D)  # one projection; q, k and v are slices of it
    fused[:, Hq * D:(Hq + Hkv) * D] += offset.reshape(-1)
    fused = fused.to(dtype)
    state["q"] = fused[:, :Hq * D].view(T, Hq, D)
    state["new_k"] = fused[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
    state["new_v"] = fused[:, (Hq + Hkv) * D:].view(T, Hkv, D)
    ends = [0]
    for _, n in seqs:
        ends.append(ends[-1] + n)
    state["lengths"] = torch.tensor([length for length, _ in seqs], dtype=torch.int32, device="cuda")
    state["starts"] = torch.tensor(ends, dtype=torch.int32, device="cuda") if T != B else None  # None: one token each
    # what is read back: whole sequences, or after a write the written tokens and those that shared their first page
    back = [length if case["kind"] == "read" else min(length, n + page - 1) for length, n in seqs]
    ends = [0]
    for n in back:
        ends.append(ends[-1] + n)
    state["back"] = back
    state["back_starts"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    state["max_length"] = max(length for length, _ in seqs)
    if own:
        from autorust_b200 import ops
        state["cache"] = ops.KvCache(state["k"], state["v"], state["k_scale"], state["v_scale"], state["k_mean"])
    return state


def _own(state):
    from autorust_b200 import ops
    case, cache = state["case"], state["cache"]
    where = (state["table"], state["lengths"])
    if case["kind"] in ("step", "write"):
        ops.kv_cache_append(cache, state["new_k"], state["new_v"], *where, state["starts"])
    out = {}
    if case["kind"] in ("step", "attend"):
        out["o"] = ops.kv_cache_attention(cache, state["q"], *where, state["starts"], causal=case["causal"],
                                          max_length=max(1, state["max_length"]))
    if case["kind"] != "attend":
        out["k"], out["v"] = ops.kv_cache_read(cache, *where, state["back_starts"], sum(state["back"]), dtype=_dtype(case))
    return out


def run(state):
    if own:
        return _own(state)
    case, page = state["case"], state["case"]["page"]
    table, mean = state["table"], state["k_mean"]
    G = case["Hq"] // case["Hkv"]
    if case["kind"] in ("step", "write"):
        row = 0
        for b, (length, n) in enumerate(state["seqs"]):
            if length >= n:
                k = state["new_k"][row:row + n].float()
                k = k - mean if mean is not None else k
                _write(state["k"], state["k_scale"], k, table[b], length - n, page, case["fp8"])
                _write(state["v"], state["v_scale"], state["new_v"][row:row + n].float(), table[b], length - n, page, case["fp8"])
            row += n
    outs, row = {name: [] for name in _outputs(case)}, 0
    for b, (length, n) in enumerate(state["seqs"]):
        k = _gather(state["k"], state["k_scale"], table[b], length, page)
        v = _gather(state["v"], state["v_scale"], table[b], length, page)
        if "k" in outs:
            back = k[length - state["back"][b]:]
            outs["k"].append((back + mean if mean is not None else back).to(_dtype(case)))
            outs["v"].append(v[length - state["back"][b]:].to(_dtype(case)))
        if "o" not in outs:
            continue
        q = state["q"][row:row + n].float()
        row += n
        if length == 0:
            outs["o"].append(torch.zeros_like(q).to(_dtype(case)))
            continue
        q = q.view(n, case["Hkv"], G, case["D"]).permute(1, 0, 2, 3).reshape(case["Hkv"], n * G, case["D"])
        s = q @ k.permute(1, 2, 0) / float(case["D"]) ** 0.5
        if case["causal"] and n > 1:
            last = torch.arange(length - n, length, device=s.device).repeat_interleave(G)
            s.masked_fill_(torch.arange(length, device=s.device)[None, None, :] > last[None, :, None], float("-inf"))
        p = torch.exp(s - s.amax(dim=-1, keepdim=True))
        o = (p @ v.permute(1, 0, 2)) / p.sum(dim=-1, keepdim=True)
        o = o.view(case["Hkv"], n, G, case["D"]).permute(1, 0, 2, 3).reshape(n, case["Hq"], case["D"])
        outs["o"].append(o.to(_dtype(case)))
    return {name: torch.cat(parts) for name, parts in outs.items()}


def work(case):
    seqs = _sequences(case)
    size = 4 if case["dtype"] == "f32" else 2
    Hq, Hkv, D, page, new = case["Hq"], case["Hkv"], case["D"], case["page"], sum(n for _, n in _sequences(case))
    token = 2 * Hkv * D  # codes of one token's key and value
    nbytes, flops = 0, 0
    if case["kind"] in ("step", "write"):  # the new keys and values in, their codes out
        nbytes += sum((size + 1) * token * n for length, n in seqs if length)
        flops += sum(3 * token * n for length, n in seqs if length)
    if case["kind"] in ("step", "attend"):
        for length, n in seqs:
            held = length - n if case["kind"] == "step" else length  # what was written in this call need not be read back
            nbytes += held * token + (length + page - 1) // page * (8 * Hkv + 4)
            pairs = sum(length - n + 1 + i for i in range(n)) if case["causal"] else n * length
            flops += 4 * D * Hq * pairs if length else 0
        nbytes += 2 * size * new * Hq * D
    if case["kind"] != "attend":
        for length, n in seqs:
            back = length if case["kind"] == "read" else min(length, n + page - 1)
            held = {"read": back, "write": back - min(back, n), "step": 0}[case["kind"]]  # a step's attention has read them
            nbytes += held * token + back * token * size + (back + page - 1) // page * (8 * Hkv + 4)
            flops += back * token
    return {"bytes": int(nbytes), "flops": int(flops)}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------
def _e4m3_values():
    """The 256 values an E4M3 code stands for, from the format: sign, 4 exponent bits with bias 7, 3 mantissa bits."""
    table = []
    for code in range(256):
        e, m = (code >> 3) & 15, code & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        table.append(float("nan") if code & 127 == 127 else (-x if code & 128 else x))
    return table


class _Exact:
    """One of the two code tensors with its scales, held in 64 bits: the codes' values and the scales, which are f32 numbers."""

    def __init__(self, codes, scales):
        self.fp8 = codes.dtype == torch.uint8
        if self.fp8:
            self.held = torch.tensor(_e4m3_values(), dtype=torch.float64, device=codes.device)[codes.long()]
        else:
            self.held = codes.double()
        self.scales = scales.double()

    @staticmethod
    def f32(x):
        return x.to(torch.float32).double()

    def nearest(self, y):
        if not self.fp8:
            return torch.round(y)
        # nearest multiple of the step of y's binade, ties to the even multiple
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
        return torch.round(y / step) * step

    def put(self, x, pages, first, page):
        """x [n, Hkv, D]: page by page."""
        end = first + x.shape[0]
        for j in range(first // page, (end - 1) // page + 1):
            lo, hi = max(first, j * page), min(end, (j + 1) * page)
            at, part = pages[j], x[lo - first:hi - first].transpose(0, 1)
            amax = part.abs().amax(dim=(1, 2))
            if self.fp8:
                step = torch.full_like(amax, FLOOR)
                for e in range(-60, 61):
                    step = torch.where(amax > 448.0 * 2.0 ** (e - 1), torch.full_like(amax, 2.0 ** e), step)
            else:
                step = self.f32(amax / 127.0).clamp_min(FLOOR)
            kept = lo - j * page
            if kept:
                before = self.scales[at]
                step = torch.maximum(step, before)
                self.held[at, :, :kept] = self.nearest(self.f32(self.held[at, :, :kept] * self.f32(before / step)[:, None, None]))
            inverse = self.f32(1.0 / step)[:, None, None]
            self.held[at, :, kept:kept + hi - lo] = self.nearest(self.f32(part * inverse))
            self.scales[at] = step

    def tokens(self, pages, length, page):
        n = (length + page - 1) // page
        at = torch.tensor(pages[:n], dtype=torch.long, device=self.held.device)
        x = self.held[at] * self.scales[at][:, :, None, None]
        return x.transpose(1, 2).flatten(0, 1)[:length]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    page, G, mean = case["page"], case["Hq"] // case["Hkv"], state["k_mean"]
    keys, values = _Exact(state.pop("k"), state["k_scale"]), _Exact(state.pop("v"), state["v_scale"])
    table = state["table"].tolist()
    row, outs = 0, {name: [] for name in _outputs(case)}
    for pages, (length, n), back in zip(table, state["seqs"], state["back"]):
        rows = slice(row, row + n)
        row += n
        if case["kind"] in ("step", "write") and length >= n:
            k = state["new_k"][rows].double()
            keys.put(_Exact.f32(k - mean.double()) if mean is not None else k, pages, length - n, page)
            values.put(state["new_v"][rows].double(), pages, length - n, page)
        if "k" in outs:
            k = keys.tokens(pages, length, page)
            k = k + mean.double() if mean is not None else k
            outs["k"].append(k[length - back:])
            outs["v"].append(values.tokens(pages, length, page)[length - back:])
        if "o" not in outs:
            continue
        o = torch.zeros(n, case["Hq"], case["D"], dtype=torch.float64, device="cuda")
        if length:
            k, v = keys.tokens(pages, length, page), values.tokens(pages, length, page)
            q = state["q"][rows].double()
            hidden = None
            if case["causal"]:
                hidden = torch.arange(length, device="cuda")[None, :] > torch.arange(length - n, length, device="cuda")[:, None]
            for h in range(case["Hq"]):
                logits = q[:, h] @ k[:, h // G].T * case["D"] ** -0.5
                if hidden is not None:
                    logits = logits.masked_fill(hidden, -float("inf"))
                o[:, h] = torch.softmax(logits, dim=-1) @ v[:, h // G]
        outs["o"].append(o)
    return {name: torch.cat(parts) for name, parts in outs.items()}
