"""The short and the long host path take and refuse the same calls: every argument of append, read and attend in turn is replaced by
forms that are odd or wrong, and both ways have to give the same bits or the same exception."""
import numpy as np
import pytest
import torch

from mimo_stream import KVCache, PageTable, Rotary, StepPlan, append, attend, read

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
E4M3 = torch.float8_e4m3fn
HEADS, KV, D, PAGE, N = 4, 2, 64, 16, 21


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _apart(t):
    """The same values with a gap behind each of the last dimension's."""
    return torch.stack((t, t), -1)[..., 0]


def _unaligned(t):
    return torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


def _far(t):
    """The same rows at twice the distance."""
    return torch.cat((t, t), 1)[:, :t.shape[1]] if t.dim() > 1 else torch.stack((t, t), 1)[:, 0]


TENSOR_FORMS = {"none": lambda t: None, "cpu": lambda t: t.cpu(), "int64": lambda t: t.long(), "float": lambda t: t.float(), "half": lambda t: t.half(),
                "double": lambda t: t.double(), "short": lambda t: t[:-1], "first": lambda t: t[:1], "empty": lambda t: t[:0], "deeper": lambda t: t[None],
                "flat": lambda t: t.reshape(-1), "apart": _apart, "unaligned": _unaligned, "far": _far, "narrow": lambda t: t[..., :-1],
                "parameter": lambda t: torch.nn.Parameter(t, requires_grad=False), "list": lambda t: t.tolist(), "one number": lambda t: t.flatten()[0],
                "swapped": lambda t: t.transpose(0, -1), "expanded": lambda t: t[:1].expand(t.shape), "turned": lambda t: t.flip(0)}
NUMBERS = [None, -1, 0, 1, 2, 7, PAGE, 32, 1 << 31, 1 << 40, 1 << 70, 0.5, 1.5, -0.25, float("nan"), float("inf"), True, "x", np.int64(3), np.float32(0.5)]


def _state(kind, shorten=True):
    if kind == "bf16":
        cache = KVCache(8, PAGE, KV, D, D)
    else:
        cache = KVCache(8, PAGE, KV, D, D, dtype=E4M3, **(dict(block_scales=True) if kind == "blocks" else dict(k_scale=0.1, v_scale=0.2)))
    rng = np.random.default_rng(3)
    plan = PageTable(2, 4, 8, PAGE).step(i32([16, 5]), N)
    q, k, v = (torch.from_numpy(rng.standard_normal((N, h, D)).astype(np.float32)).to(BF).cuda() for h in (HEADS, KV, KV))
    append(cache, plan, k, v)
    attend(q, cache, plan)                                 # the stream's workspace is there
    if not shorten:
        cache._call = None
    given = dict(slots=plan.slots, positions=plan.positions, status=torch.zeros(1, dtype=torch.int32, device="cuda"), page_size=PAGE, starts=plan.starts,
                 lens=plan.lens, table=plan.table, max_new=16, k=k, v=v, q=q, scale=0.125, window=0, sink_tokens=0,
                 sink_logits=torch.zeros(HEADS, device="cuda"), out=torch.zeros(N, HEADS, D, dtype=BF, device="cuda"), rotary=Rotary(32))
    return cache, given


def _append(cache, g):
    return append(cache, StepPlan(slots=g["slots"], positions=g["positions"], status=g["status"], page_size=g["page_size"]), g["k"], g["v"], q=g["q"], rotary=g["rotary"])


def _read(cache, g):
    return read(cache, g["slots"], status=g["status"])


def _attend(cache, g):
    plan = StepPlan(starts=g["starts"], lens=g["lens"], table=g["table"], max_new=g["max_new"], status=g["status"], page_size=g["page_size"])
    return attend(g["q"], cache, plan, g["scale"], g["window"], g["sink_tokens"], g["sink_logits"], g["out"])


CALLS = {"append": (_append, ["slots", "positions", "status", "k", "v", "q"], ["page_size"]),
         "read": (_read, ["slots", "status"], []),
         "attend": (_attend, ["q", "starts", "lens", "table", "status", "sink_logits", "out"], ["page_size", "max_new", "scale", "window", "sink_tokens"])}


def _outcome(call, kind, shorten, change):
    cache, given = _state(kind, shorten)
    name, form = change
    try:
        given[name] = form(given[name])
    except (RuntimeError, IndexError, ValueError, TypeError):
        return "no such form"
    try:
        got = call(cache, given)
    except Exception as e:                                 # noqa: BLE001 (which one is what is compared)
        torch.cuda.synchronize()
        return type(e), str(e)
    tensors = [] if got is None else list(got) if isinstance(got, tuple) else [got]
    held = [cache.k.view(torch.uint8), cache.v.view(torch.uint8)]
    status = given["status"]
    return [t.detach().cpu().view(torch.uint8) for t in (*tensors, *held)], status.tolist() if isinstance(status, torch.Tensor) else None


def _same(a, b):
    if isinstance(a, tuple) and isinstance(a[0], list) and isinstance(b, tuple) and isinstance(b[0], list):
        return a[1] == b[1] and len(a[0]) == len(b[0]) and all(torch.equal(x, y) for x, y in zip(a[0], b[0]))
    return not isinstance(a[0], list) and not isinstance(b[0], list) and a == b


@pytest.mark.parametrize("kind", ["bf16", "heads", "blocks"])
@pytest.mark.parametrize("name", list(CALLS))
def test_both_ways_have_one_rule(name, kind):
    call, tensors, numbers = CALLS[name]
    changes = [(t, f"{t} {label}", form) for t in tensors for label, form in TENSOR_FORMS.items()]
    changes += [(n, f"{n} {value!r}", lambda _, value=value: value) for n in numbers for value in NUMBERS]
    if name == "append":
        changes += [("rotary", f"rotary {r}", lambda _, make=make: make()) for r, make in
                    (("none", lambda: None), ("cpu", lambda: Rotary(32, device="cpu")), ("wide", lambda: Rotary(128)), ("side", lambda: Rotary(64, interleaved=True)))]
    differ = [label for arg, label, form in changes if not _same(*(_outcome(call, kind, shorten, (arg, form)) for shorten in (True, False)))]
    assert not differ
