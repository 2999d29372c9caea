"""The adapters' formula in 64 bits on the host, and how far a kernel's sums may be from it."""
import torch


def reference(out, x, adapters, slots):
    """(out + the adapters' part, the sum of the magnitudes that enter it) in 64 bits; `out`, `x`, `a`, `b`,
    `scales`, `ranks` and `slots` on the host. Rows without an adapter: out itself, magnitude 0."""
    a, b, scales, ranks = adapters
    want, size = out.double().clone(), torch.zeros_like(out, dtype=torch.float64)
    for m, s in enumerate(slots.tolist()):
        if not 0 <= s < a.shape[0]:
            continue
        r = max(0, min(a.shape[1], a.shape[1] if ranks is None else int(ranks[s])))
        scale = 1.0 if scales is None else float(scales[s])
        xs, aa, bb = x[m].double(), a[s, :r].double(), b[s, :, :r].double()
        want[m] += scale * (bb @ (aa @ xs))
        size[m] = abs(scale) * (bb.abs() @ (aa.abs() @ xs.abs()))
    return want, size


def bound(want, size, out, inner, rank):
    """Half a step of out's type on the result, and of the magnitudes that enter: 2^-24 for each of the
    additions in fp32 behind a value (inner terms, then up to three pieces of `rank` terms), and what the
    pieces of the first products leave of them, 2^-16 (two pieces of bf16, half a step 2^-8 each) for a
    bf16 result and 2^-24 (three pieces) for fp32."""
    pieces = 2.0 ** -24 if out.dtype == torch.float32 else 2.0 ** -16
    half = torch.finfo(out.dtype).eps / 2
    sums = size * ((inner + 3 * rank + 64) * 2.0 ** -24 + pieces)
    return half * (want.abs() + sums) + sums


def check(got, before, x, adapters, slots, label=""):
    """`got` (device) is `before` (host) plus the adapters' part; rows without one are untouched bits."""
    want, size = reference(before, x, adapters, slots)
    a = adapters[0]
    tol = bound(want, size, before, a.shape[2], a.shape[1])
    got = got.cpu()
    off = (got.double() - want).abs() - tol
    assert off.max() <= 0, f"{label}: {off.max().item()} past the bound at {divmod(int(off.argmax()), got.shape[1])}"
    idle = (size == 0).all(1)
    same = torch.int32 if got.dtype == torch.float32 else torch.int16
    assert torch.equal(got[idle].contiguous().view(same), before[idle].contiguous().view(same)), \
        f"{label}: a row without an adapter was written"
