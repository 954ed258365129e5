"""Performance cases: a decoding loop's operators on one GPU.

The program holds its tensors in torch and calls the C ABI through
``tensorcx_hip_capi`` with plain pointers, descriptors and one scratch buffer
that it keeps, on torch's current stream:

``window``  attention over float32 keys and values with a sliding window and
            first tokens (sinks) that stay visible, grouped heads
``store``   keys and values quantised into a 4-bit cache at each sequence's
            position, and the stored tokens read back as float32
``cache``   attention over the 4-bit cache (optionally windowed)
``step``    one decoding step: the new token stored, then attention over the cache
``select``  beam search's choice over beams and vocabulary
``reorder`` the states moved to the chosen beams

A case is a dict of plain values; ``kind`` picks the path. Where ``own`` is
false, ``run`` computes the same in elementary torch operations.
"""

from __future__ import annotations

import math
import pathlib
import sys

import numpy as np
import torch

own = False

GROUP = 32  # features that share a scale word

# No drawn case does more than the largest listed ones.
MAX_BYTES = 1.68e8
MAX_FLOPS = 6e10
MAX_SCORES = 5e9  # bytes of the score matrix that the plain form holds


def listed():
    return [
        # One new token for each of eight sequences of different lengths; 32 query heads on 8 cached ones.
        {"name": "window_decode", "kind": "window", "batch": 8, "heads": 32, "kv_heads": 8, "rows": 1, "cols": 8192,
         "features": 128, "window": 1024, "sinks": 4, "ragged": True},
        # A prompt; the window is a quarter of it.
        {"name": "window_prompt", "kind": "window", "batch": 1, "heads": 16, "kv_heads": 4, "rows": 4096, "cols": 4096,
         "features": 128, "window": 1024, "sinks": 4, "ragged": False},
        # A long prompt with narrow heads, one for one.
        {"name": "window_prompt_long", "kind": "window", "batch": 1, "heads": 16, "kv_heads": 16, "rows": 8192,
         "cols": 8192, "features": 64, "window": 2048, "sinks": 16, "ragged": False},
        # A few more tokens of short padded sequences, sizes that fit no tile.
        {"name": "window_chunk_odd", "kind": "window", "batch": 3, "heads": 6, "kv_heads": 2, "rows": 37, "cols": 301,
         "features": 80, "window": 50, "sinks": 3, "ragged": True},
        # A prompt's keys and values into the cache.
        {"name": "store_prompt", "kind": "store", "batch": 2, "kv_heads": 8, "rows": 4096, "cols": 5000, "features": 128},
        # One step of a short chat: latency.
        {"name": "step_short", "kind": "step", "batch": 1, "heads": 8, "kv_heads": 8, "rows": 1, "cols": 512,
         "features": 64, "window": 0, "sinks": 0, "ragged": False},
        # Sixteen sequences of up to 8192 tokens, grouped heads.
        {"name": "cache_decode", "kind": "cache", "batch": 16, "heads": 32, "kv_heads": 8, "rows": 1, "cols": 8192,
         "features": 128, "window": 0, "sinks": 0, "ragged": True},
        # One very long sequence, a head for a head.
        {"name": "cache_decode_long", "kind": "cache", "batch": 1, "heads": 16, "kv_heads": 16, "rows": 1,
         "cols": 131072, "features": 64, "window": 0, "sinks": 0, "ragged": False},
        # Beams of a small batch over a usual vocabulary.
        {"name": "select_small", "kind": "select", "batch": 1, "beams": 4, "vocabulary": 32000, "count": 4, "finished": True},
        # A large batch over a large vocabulary, twice as many candidates as beams.
        {"name": "select_large", "kind": "select", "batch": 16, "beams": 8, "vocabulary": 128256, "count": 16,
         "finished": False},
        # A layer's 4-bit caches follow their beams; and a wide float32 state.
        {"name": "reorder_caches", "kind": "reorder", "batch": 4, "beams": 4, "count": 4, "tensors": 2,
         "row_words": 8 * 1024 * 20, "dtype": "int32"},
        {"name": "reorder_states", "kind": "reorder", "batch": 16, "beams": 8, "count": 8, "tensors": 4,
         "row_words": 4101, "dtype": "float32"},
    ]


# ------------------------------------------------------------------ drawing
def _size(rng, low, high):
    """Spread over the logarithm of [low, high]; one in three a multiple of 64."""
    value = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.33 and value >= 96:
        value = (value + 32) // 64 * 64
    return max(low, min(high, value))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 8, 16])
    return kv * rng.choice([1, 1, 2, 4, 5, 8]), kv


def _draw_window(rng):
    heads, kv = _heads(rng)
    cols = _size(rng, 1, 16384)
    rows = rng.choice([1, 1, min(cols, _size(rng, 2, 64)), cols])
    return {"kind": "window", "batch": _size(rng, 1, 16), "heads": heads, "kv_heads": kv, "rows": rows, "cols": cols,
            "features": rng.choice([32, 64, 64, 80, 128, 128]), "window": rng.choice([0, _size(rng, 1, 4096), _size(rng, 1, 4096)]),
            "sinks": rng.choice([0, 1, 4, 4, 70]), "ragged": rows < cols and rng.random() < 0.7}


def _draw_cache(rng, kind):
    heads, kv = _heads(rng)
    cols = _size(rng, 16, 131072)
    return {"kind": kind, "batch": _size(rng, 1, 32), "heads": heads, "kv_heads": kv,
            "rows": 1 if kind == "step" else rng.choice([1, 1, 1, min(cols, _size(rng, 2, 40))]), "cols": cols,
            "features": rng.choice([32, 64, 128, 128]), "window": rng.choice([0, 0, _size(rng, 1, 4096)]),
            "sinks": rng.choice([0, 1, 4, 70]), "ragged": rng.random() < 0.7}


def _draw_store(rng):
    cols = _size(rng, 1, 16384)
    return {"kind": "store", "batch": _size(rng, 1, 8), "kv_heads": rng.choice([1, 2, 3, 8, 16]), "rows": _size(rng, 1, cols),
            "cols": cols, "features": rng.choice([32, 64, 128])}


def _draw_select(rng):
    beams, vocabulary = rng.choice([1, 2, 3, 4, 5, 8, 16]), _size(rng, 64, 150000)
    return {"kind": "select", "batch": _size(rng, 1, 32), "beams": beams, "vocabulary": vocabulary,
            "count": rng.choice([1, beams, 2 * beams, 2 * beams]), "finished": rng.random() < 0.4}


def _draw_reorder(rng):
    beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
    return {"kind": "reorder", "batch": _size(rng, 1, 32), "beams": beams, "count": rng.choice([1, beams, beams]),
            "tensors": rng.randint(1, 10), "row_words": _size(rng, 1, 300000), "dtype": rng.choice(["float32", "int32"])}


def draw(rng):
    """One more case of the listed kinds; sizes too large for one pass are drawn again."""
    pick = rng.choice([_draw_window, _draw_window, lambda r: _draw_cache(r, "cache"), lambda r: _draw_cache(r, "cache"),
                       lambda r: _draw_cache(r, "step"), _draw_store, _draw_select, _draw_reorder])
    while True:
        case = pick(rng)
        needs = work(case)
        scores = 4 * case["batch"] * case["heads"] * case["rows"] * case["cols"] if "heads" in case else 0
        dense = 4 * case["batch"] * case["kv_heads"] * case["cols"] * case["features"] if "cols" in case else 0
        if needs["bytes"] <= MAX_BYTES and needs["flops"] <= MAX_FLOPS and max(scores, 2 * dense) <= MAX_SCORES:
            return case


# ------------------------------------------------------------------ sizes
def _lengths(case):
    """Tokens of each sequence: all of cols, or spread from half of them up."""
    batch, cols = case["batch"], case["cols"]
    if not case.get("ragged"):
        return [cols] * batch
    return [max(1, cols - (b * (cols // 2)) // batch - b) for b in range(batch)]


def _visible(case, length):
    """For each query of a sequence of that length, the keys it sees; and the keys that any of them sees."""
    rows, window, sinks = case["rows"], case["window"], case["sinks"]
    p = np.arange(length - rows, length, dtype=np.int64)
    if window == 0:
        seen = np.maximum(p + 1, 0)
        return int(seen.sum()), max(length, 0)
    first = np.maximum(p - window + 1, 0)
    seen = np.where(p >= 0, p + 1 - first + np.minimum(sinks, first), 0)
    low = max(int(p[0]) - window + 1, 0)
    return int(seen.sum()), max(length, 0) - low + min(sinks, low)


def work(case):
    """Bytes (each input read once, each output written once) and operations of one pass."""
    kind = case["kind"]
    if kind == "select":
        n = case["batch"] * case["beams"]
        return {"bytes": 4 * n * case["vocabulary"] + 5 * n + 12 * case["batch"] * case["count"],
                "flops": 3 * n * case["vocabulary"]}
    if kind == "reorder":
        rows = case["batch"] * case["count"]
        return {"bytes": case["tensors"] * 8 * rows * case["row_words"] + 4 * rows, "flops": 0}
    features = case["features"]
    token = features // 2 + features // 8  # bytes of a cached token and head
    if kind == "store":  # tokens read as float32 and stored; the cache read and written as float32; keys and values
        lead = case["batch"] * case["kv_heads"]
        return {"bytes": 2 * lead * (case["rows"] + case["cols"]) * (4 * features + token) + 4 * case["batch"],
                "flops": 2 * lead * (6 * case["rows"] + 2 * case["cols"]) * features}
    pairs, keys = 0, 0
    for length in _lengths(case):
        seen, touched = _visible(case, length)
        pairs, keys = pairs + seen, keys + touched
    io = 8 * case["batch"] * case["heads"] * case["rows"] * features + 4 * case["batch"]
    per_key = 8 * features if kind == "window" else 2 * token
    more = 2 * case["batch"] * case["kv_heads"] * 4 * features if kind == "step" else 0
    return {"bytes": io + keys * case["kv_heads"] * per_key + more, "flops": 4 * features * case["heads"] * pairs}


# ------------------------------------------------------------------ the 4-bit format
def _quantise(x):
    """(..., features) float32 to codes (..., features) and scale words (..., features / 32). Of each 32
    features: the low end rounded down to bfloat16, the step (max - low) / 15 rounded up to it."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    low, high = g.amin(-1) + 0.0, g.amax(-1)
    bits = low.view(torch.int32)
    cut = bits & -65536
    low_bits = torch.where((cut != bits) & (bits < 0), cut + 65536, cut)
    low = low_bits.view(torch.float32)
    bits = ((high - low) * torch.tensor(1.0 / 15.0, dtype=torch.float32, device=x.device)).view(torch.int32)
    cut = bits & -65536
    step_bits = torch.where(cut != bits, cut + 65536, cut)
    step = step_bits.view(torch.float32)
    codes = torch.round((g - low[..., None]) / step[..., None])
    codes = torch.where(step[..., None] > 0, codes, torch.zeros_like(codes)).clamp(0, 15).to(torch.int32)
    return codes.reshape(x.shape), low_bits | ((step_bits >> 16) & 65535)


def _pack(x):
    """Cache rows: byte n (features / 32) + g of the codes holds features 32 g + n and (in its high half)
    32 g + 16 + n; the scale words follow."""
    codes, words = _quantise(x)
    groups = x.shape[-1] // GROUP
    c = codes.reshape(*x.shape[:-1], groups, 2, 16)
    data = (c[..., 0, :] | (c[..., 1, :] << 4)).transpose(-1, -2).contiguous().to(torch.uint8)
    data = data.reshape(*x.shape[:-1], x.shape[-1] // 2).view(torch.int32)
    return torch.cat([data, words], -1)


def _unpack(rows, features, dtype=torch.float32):
    """Cache rows to the values they stand for."""
    groups = features // GROUP
    data = rows[..., :features // 8].contiguous().view(torch.uint8).reshape(*rows.shape[:-1], 16, groups)
    data = data.transpose(-1, -2).to(torch.int32)
    codes = torch.cat([data & 15, data >> 4], -1).to(dtype)
    words = rows[..., features // 8:].contiguous()
    low = (words & -65536).view(torch.float32).to(dtype)
    step = (words << 16).view(torch.float32).to(dtype)
    return (low[..., None] + step[..., None] * codes).reshape(*rows.shape[:-1], features)


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=generator, device="cuda") * scale

    def integers(low, high, shape):
        return torch.randint(low, high, shape, generator=generator, device="cuda", dtype=torch.int32)

    kind = case["kind"]
    if kind == "select":
        batch, beams = case["batch"], case["beams"]
        t = {"logits": normal(batch, beams, case["vocabulary"], scale=3.0), "scores": normal(batch, beams, scale=2.0) - 20.0}
        if case["finished"]:
            t["finished"] = integers(0, 4, (batch, beams)) == 0
        return t
    if kind == "reorder":
        rows = case["batch"] * case["beams"]
        make = normal if case["dtype"] == "float32" else lambda *shape: integers(-2 ** 31, 2 ** 31 - 1, shape)
        return {"states": [make(rows, case["row_words"]) for _ in range(case["tensors"])],
                "beams": integers(0, case["beams"], (case["batch"], case["count"]))}
    batch, kv, rows, cols, features = (case[n] for n in ("batch", "kv_heads", "rows", "cols", "features"))

    def keys(n):  # keys have features of a level of their own
        return normal(batch, kv, n, features) + normal(1, kv, 1, features, scale=2.0)

    if kind == "store":
        positions = integers(0, cols - rows + 1, (batch,))
        return {"key": keys(rows), "value": normal(batch, kv, rows, features), "positions": positions}
    order = torch.randperm(batch, generator=generator, device="cuda")
    t = {"query": normal(batch, case["heads"], rows, features),
         "lengths": torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order]}
    if kind == "window":
        t["key"], t["value"] = keys(cols), normal(batch, kv, cols, features)
        return t
    if kind == "step":
        t["positions"] = t["lengths"] - 1
        t["key"], t["value"] = keys(1), normal(batch, kv, 1, features)
    # The cache as the steps before left it: of a few distinct tokens, so that making it is quick.
    distinct = min(cols, 4096)
    repeat = (cols + distinct - 1) // distinct
    t["key_cache"] = _pack(keys(distinct)).repeat(1, 1, repeat, 1)[:, :, :cols].contiguous()
    t["value_cache"] = _pack(normal(batch, kv, distinct, features)).repeat(1, 1, repeat, 1)[:, :, :cols].contiguous()
    return t


def prepare(case, seed):
    """The inputs, and the outputs and the scratch memory that the program keeps."""
    t, kind = _inputs(case, seed), case["kind"]
    state = {"case": dict(case), "tensors": t, "plan": {}, "scratch": torch.empty(32 << 20, dtype=torch.uint8, device="cuda")}

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="cuda")

    if kind == "select":
        shape = (case["batch"], case["count"])
        state["out"] = [empty(*shape), empty(*shape, dtype=torch.int32), empty(*shape, dtype=torch.int32)]
    elif kind == "reorder":
        rows = case["batch"] * case["count"]
        state["out"] = [empty(rows, case["row_words"], dtype=s.dtype) for s in t["states"]]
    elif kind == "store":
        words = case["features"] // 8 + case["features"] // GROUP
        shape = (case["batch"], case["kv_heads"], case["cols"], words)
        t["key_cache"], t["value_cache"] = (torch.zeros(shape, dtype=torch.int32, device="cuda") for _ in range(2))
        state["out"] = [empty(case["batch"], case["kv_heads"], case["cols"], case["features"]) for _ in range(2)]
    else:
        state["out"] = empty(case["batch"], case["heads"], case["rows"], case["features"])
    return state


# ------------------------------------------------------------------ the framework's operators
def _capi():
    path = str(pathlib.Path(__file__).resolve().parents[1] / "tensor.cx_amd" / "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import tensorcx_hip_capi as capi
    return capi


def _attention_plan(capi, case, t, state):
    return capi.window_attention_desc(case["batch"], case["heads"], case["kv_heads"], case["rows"], case["cols"],
                                      case["features"], window=case["window"], sinks=case["sinks"],
                                      scale=case["features"] ** -0.5, lengths=t["lengths"].data_ptr())


def _store_plan(capi, case):
    return capi.cache4_store_desc(case["batch"], case["kv_heads"], case["rows"], case["cols"], case["features"])


def _own(state):
    case, t, plan, out = state["case"], state["tensors"], state["plan"], state["out"]
    kind, stream = case["kind"], torch.cuda.current_stream().cuda_stream
    if not plan:  # what the program keeps from call to call
        capi = plan["capi"] = _capi()
        wanted = 0  # the scratch buffer, or one of the size that the library asks for where that is more
        if kind in ("window", "cache", "step"):
            plan["desc"] = _attention_plan(capi, case, t, state)
            wanted = capi.window_attention_workspace_bytes(plan["desc"], cache=kind != "window")
        elif kind == "select":
            wanted = capi.beam_select_workspace_bytes(case["batch"], case["beams"], case["vocabulary"], case["count"])
        plan["scratch"] = state["scratch"] if wanted <= state["scratch"].numel() else torch.empty(
            wanted, dtype=torch.uint8, device="cuda")
        plan["workspace"] = capi.Workspace(plan["scratch"].data_ptr(), plan["scratch"].numel())
        if kind in ("store", "step"):
            plan["store"] = _store_plan(capi, case)
        if kind == "reorder":
            plan["reorder"] = capi.beam_reorder_plan([s.data_ptr() for s in t["states"]], [o.data_ptr() for o in out],
                                                     [4 * case["row_words"]] * case["tensors"])
    capi, workspace = plan["capi"], plan["workspace"]
    if kind == "window":
        capi.window_attention(t["query"].data_ptr(), t["key"].data_ptr(), t["value"].data_ptr(), out.data_ptr(),
                              plan["desc"], workspace=workspace, s=stream)
        return out
    if kind == "select":
        finished = t["finished"].data_ptr() if case["finished"] else None
        capi.beam_select(t["logits"].data_ptr(), t["scores"].data_ptr(), out[0].data_ptr(), out[1].data_ptr(),
                         out[2].data_ptr(), case["batch"], case["beams"], case["vocabulary"], case["count"],
                         finished=finished, eos=2, workspace=workspace, s=stream)
        return out
    if kind == "reorder":
        capi.beam_reorder(plan["reorder"], t["beams"].data_ptr(), case["batch"], case["beams"], case["count"], s=stream)
        return out
    keys, values = t["key_cache"].data_ptr(), t["value_cache"].data_ptr()
    if kind in ("store", "step"):
        capi.cache4_store(t["key"].data_ptr(), t["value"].data_ptr(), keys, values, t["positions"].data_ptr(),
                          plan["store"], s=stream)
    if kind == "store":
        for cache, o in zip((keys, values), out):
            capi.cache4_load(cache, o.data_ptr(), case["batch"] * case["kv_heads"], case["cols"], 0, case["cols"],
                             case["features"], s=stream)
        return out
    capi.cache4_attention(t["query"].data_ptr(), keys, values, out.data_ptr(), plan["desc"], workspace=workspace,
                          s=stream)
    return out


# ------------------------------------------------------------------ the plain form
def _attend(case, query, key, value, lengths):
    """Scores of all pairs, the visible ones' softmax, the values' sum."""
    batch, kv, rows, cols = case["batch"], case["kv_heads"], case["rows"], case["cols"]
    q = query.reshape(batch, kv, -1, case["features"])
    scores = torch.matmul(q, key.transpose(-1, -2)) * case["features"] ** -0.5
    scores = scores.reshape(batch, case["heads"], rows, cols)
    j = torch.arange(cols, device=query.device)
    p = lengths.long()[:, None] - rows + torch.arange(rows, device=query.device)
    seen = j <= p[..., None]
    if case["window"]:
        seen = seen & ((j > p[..., None] - case["window"]) | (j < case["sinks"]))
    seen = seen[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    weights = (weights / torch.where(total == 0, torch.ones_like(total), total)).reshape(batch, kv, -1, cols)
    return torch.matmul(weights, value).reshape(query.shape)


def _slots(positions, rows):
    return positions.long()[:, None] + torch.arange(rows, device=positions.device)


def _store(cache, x, positions):
    batch = torch.arange(x.shape[0], device=x.device)[:, None]
    cache[batch, :, _slots(positions, x.shape[2])] = _pack(x).transpose(1, 2)


def _select(case, logits, scores, finished):
    """In 64 bits: neighbours in the order are as near as the logits' last bits."""
    vocabulary = case["vocabulary"]
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    total = torch.exp(x - top).sum(-1, keepdim=True)
    x = x - (top + torch.log(total)) + scores.double()[..., None]
    if finished is not None:
        end = torch.full_like(x, -math.inf)
        end[..., 2] = scores.double()
        x = torch.where(finished[..., None], end, x)
    values, order = torch.sort(x.reshape(case["batch"], -1), dim=-1, descending=True, stable=True)
    values, order = values[:, :case["count"]], order[:, :case["count"]]
    return [values, (order // vocabulary).int(), (order % vocabulary).int()]


def _plain(state):
    case, t = state["case"], state["tensors"]
    kind = case["kind"]
    if kind == "window":
        return _attend(case, t["query"], t["key"], t["value"], t["lengths"])
    if kind == "select":
        values, beams, tokens = _select(case, t["logits"], t["scores"], t.get("finished"))
        return [values.float(), beams, tokens]
    if kind == "reorder":
        rows = torch.arange(case["batch"], device="cuda")[:, None] * case["beams"] + t["beams"]
        return [s[rows.reshape(-1)] for s in t["states"]]
    if kind in ("store", "step"):
        _store(t["key_cache"], t["key"], t["positions"])
        _store(t["value_cache"], t["value"], t["positions"])
    key, value = _unpack(t["key_cache"], case["features"]), _unpack(t["value_cache"], case["features"])
    if kind == "store":
        return [key, value]
    return _attend(case, t["query"], key, value, t["lengths"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the results in 64 bits
def _exact_rows(words, features):
    """The values of packed rows, feature by feature from the bytes of the format, in float64."""
    data = words.contiguous().view(torch.uint8)
    out = torch.empty(*words.shape[:-1], features, dtype=torch.float64, device=words.device)
    for f in range(features):
        g = f // GROUP
        byte = data[..., f % 16 * (features // GROUP) + g].long()
        code = byte // 16 if f % GROUP >= 16 else byte % 16
        word = words[..., features // 8 + g]
        low = (word // 65536 * 65536).view(torch.float32).double()
        out[..., f] = low + (word * 65536).view(torch.float32).double() * code
    return out


def _exact_store(x):
    """What a stored token stands for: the format's rule, each of its float32 steps rounded from 64 bits."""
    g = x.cpu().numpy().reshape(*x.shape[:-1], -1, GROUP)
    low32 = g.min(-1)
    low32 = np.where(low32 == 0, np.float32(0), low32)
    bits = low32.view(np.uint32).astype(np.int64)
    down = bits // 65536 * 65536 + np.where((bits % 65536 != 0) & (low32 < 0), 65536, 0)
    low = down.astype(np.uint32).view(np.float32).astype(np.float64)
    span = (g.max(-1).astype(np.float64) - low).astype(np.float32).astype(np.float64)
    bits = (span * float(np.float32(1.0 / 15.0))).astype(np.float32).view(np.uint32).astype(np.int64)
    step = ((bits + 65535) // 65536 * 65536).astype(np.uint32).view(np.float32).astype(np.float64)
    off = (g.astype(np.float64) - low[..., None]).astype(np.float32).astype(np.float64)
    codes = np.rint((off / np.where(step > 0, step, 1.0)[..., None]).astype(np.float32))
    codes = np.where(step[..., None] > 0, np.clip(codes, 0, 15), 0.0)
    return torch.from_numpy((low[..., None] + step[..., None] * codes).reshape(x.shape)).cuda()


def _exact_attention(case, query, key, value, lengths):
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    share = case["heads"] // case["kv_heads"]
    for b, n in enumerate(lengths.tolist()):
        for h in range(case["heads"]):
            k, v = key[b, h // share, :n].double(), value[b, h // share, :n].double()
            for r in range(0, case["rows"], 2048):
                q = query[b, h, r:r + 2048].double()
                p = torch.arange(r, r + q.shape[0], device=q.device)[:, None] + (n - case["rows"])
                j = torch.arange(n, device=q.device)[None]
                hidden = (j > p) | (((j <= p - case["window"]) & (j >= case["sinks"])) if case["window"] else (j < 0))
                s = (q @ k.T / math.sqrt(case["features"])).masked_fill(hidden, -math.inf)
                w = torch.softmax(s, -1).masked_fill(hidden, 0.0)
                out[b, h, r:r + 2048] = w @ v
    return out


def exact(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "reorder":
        if case["dtype"] != "float32":
            return None
        index = t["beams"].cpu().numpy()
        rows = [b * case["beams"] + int(k) for b in range(case["batch"]) for k in index[b]]
        return [s.double()[rows] for s in t["states"]]
    if kind == "select":
        x = t["logits"].double()
        x = torch.log_softmax(x, -1) + t["scores"].double().unsqueeze(-1)
        if case["finished"]:
            x[t["finished"]] = -math.inf
            x[..., 2] = torch.where(t["finished"], t["scores"].double(), x[..., 2])
        values = x.flatten(1).topk(case["count"], -1).values
        return [values, None, None]
    if kind == "window":
        return _exact_attention(case, t["query"], t["key"], t["value"], t["lengths"])
    features = case["features"]
    if kind == "store":
        found = []
        for name in ("key", "value"):
            out = torch.zeros(case["batch"], case["kv_heads"], case["cols"], features, dtype=torch.float64, device="cuda")
            stored = _exact_store(t[name])
            for b, p in enumerate(t["positions"].tolist()):
                out[b, :, p:p + case["rows"]] = stored[b]
            found.append(out)
        return found
    key, value = (_exact_rows(t[name], features) for name in ("key_cache", "value_cache"))
    if kind == "step":
        for cache, name in ((key, "key"), (value, "value")):
            stored = _exact_store(t[name])
            for b, p in enumerate(t["positions"].tolist()):
                cache[b, :, p] = stored[b, :, 0]
    return _exact_attention(case, t["query"], key, value, t["lengths"])
