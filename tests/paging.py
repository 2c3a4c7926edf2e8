"""Inputs and plain 64-bit forms shared by the tests of the paged operators."""
import torch

D_QK, D_V, PAGE = 576, 512, 64


def pages(n):
    return -(-n // PAGE)


def ints(v, device):
    return torch.tensor(v, dtype=torch.int32, device=device)


def starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def paged(lens, device, seed=0, spare=3, scale=0.5, fill=float("nan")):
    """A bf16 pool whose pages lie in a random order, `fill` wherever no sequence has a token, its table (-1 where a
    sequence has no page) and the sequences' rows."""
    g = torch.Generator().manual_seed(seed)
    total = sum(pages(n) for n in lens) + spare
    order = torch.randperm(total, generator=g).tolist()
    pool = torch.full((total, PAGE, D_QK), fill, dtype=torch.bfloat16)
    table = torch.full((len(lens), max(1, max(pages(n) for n in lens))), -1, dtype=torch.int32)
    rows, at = [], 0
    for b, n in enumerate(lens):
        x = (torch.randn(n, D_QK, generator=g) * scale).to(torch.bfloat16)
        rows.append(x)
        for j in range(pages(n)):
            table[b, j] = order[at]
            part = x[PAGE * j:PAGE * (j + 1)]
            pool[order[at], :len(part)] = part
            at += 1
    return pool.to(device), table.to(device), rows


def attention64(q, keys, ends, scale):
    """q [n, H, 576] over keys [N, 576], query i over the first ends[i]: o, lse, and sum_j w_j |v_j| and the largest
    sum_d |q_d k_d| scale, what the tolerances count, in float64 on the CPU."""
    n, H, _ = q.shape
    o = torch.zeros(n, H, D_V, dtype=torch.float64)
    a = torch.zeros(n, H, D_V, dtype=torch.float64)
    lse = torch.full((n, H), float("-inf"), dtype=torch.float64)
    top = torch.zeros(n, H, dtype=torch.float64)
    q, keys = q.double().cpu(), keys.double().cpu()
    for i in range(n):
        k = keys[:max(0, ends[i])]
        if len(k) == 0:
            continue
        x = q[i] @ k.T * scale
        lse[i] = torch.logsumexp(x, dim=1)
        w = torch.exp(x - lse[i][:, None])
        o[i], a[i] = w @ k[:, :D_V], w @ k[:, :D_V].abs()
        top[i] = (q[i].abs() @ k.abs().T).amax(1) * scale
    return o, lse, a, top


def assert_attention(o, lse, ref, what=""):
    """A score is a sum of 576 products in fp32, off by at most 600 x 2^-24 of their magnitudes' sum (d); a weight by
    2 d, the fp32 sums and exponentials by 2^-16 together; P and the output are rounded to bf16, half a step of
    2^-8 each."""
    ro, rl, a, top = ref
    d = 600 * 2.0 ** -24 * top
    tol = 2.0 ** -8 * ro.abs() + (2.0 ** -8 + 2.0 ** -16 + 2 * d[..., None]) * a
    err = (o.double().cpu() - ro).abs()
    assert torch.isfinite(o).all(), f"{what}: not finite"
    assert (err <= tol + 1e-30).all(), f"{what}: o off by {(err / (tol + 1e-30)).max().item():.3f} of the tolerance"
    dead = rl == float("-inf")
    l64 = lse.double().cpu()
    assert torch.equal(l64 == float("-inf"), dead), f"{what}: empty queries"
    el = (l64 - rl).abs()[~dead]
    tl = (d + 2.0 ** -20 * (1 + rl.abs()))[~dead]
    assert (el <= tl).all(), f"{what}: lse off by {(el / tl).max().item():.3f} of the tolerance"
