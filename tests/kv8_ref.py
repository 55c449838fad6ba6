"""The 8-bit KV cache in plain torch at 64 bits: what the GPU tests compare with, and the bounds of
their comparisons."""
import math

import torch

D, B = 128, 64
E16, E32 = 2.0 ** -11, 2.0 ** -24  # half a step of fp16 and of fp32, relative


def tree(M, rng=None):
    """Parents of a random tree (rng) or a chain (None)."""
    return [-1] + [i - 1 if rng is None else int(rng.integers(max(0, i - 5), i)) for i in range(1, M)]


def sees(parents, M):
    """[M][M]: the pass rows that each row attends (its ancestors and itself), and the depths."""
    ok, depth = torch.eye(M, dtype=torch.bool), [0] * M
    for r in range(1, M):
        p = r - 1 if parents is None else parents[r]
        ok[r] |= ok[p]
        depth[r] = depth[p] + 1
    return ok, depth


def seal(x):
    """Codes (float64 whole numbers) and scales (fp32) of blocks [..., 64, 128] fp16: each operation
    of the definition in 64 bits, rounded to the 32 it is held in."""
    x = x.double()
    a = torch.where(x.abs() < math.inf, x.abs(), torch.zeros_like(x)).amax((-2, -1))
    s = (a / torch.full_like(a, 127.0)).float()
    r = torch.where(a > 0, 127.0 / a, torch.zeros_like(a)).float()[..., None, None]
    c = (x * r.double()).float().round().clamp(-127, 127)
    c = torch.where(x.isnan() | (r == 0), torch.zeros_like(c), c)
    return c.double(), s


def page_bytes(codes, is_k):
    """[..., 64, 128] codes in the order of a page's bytes."""
    t = torch.arange(B)[:, None].expand(B, D)
    d = torch.arange(D)[None].expand(B, D)
    if is_k:
        at = 2048 * (t // 16) + 1024 * (d // 64) + 256 * (d // 16 % 4) + 16 * (t % 16) + d % 16
    else:
        at = 1024 * (d // 16) + 256 * (t // 4 % 4) + 16 * (d % 16) + 4 * (t // 16) + t % 4
    out = torch.empty(codes.shape[:-2] + (B * D,), dtype=torch.uint8, device=codes.device)
    out[..., at.reshape(-1).to(codes.device)] = (codes + 128).to(torch.uint8).flatten(-2)
    return out


def attention(q, k, v, ok):
    """softmax(q k^T / sqrt(128)) v of rows q [R, D] over keys k, v [T, D] that ok [R, T] allows (rows
    without any: zeros), the weights, and the bound of the kernel's error: its weights and outputs
    are rounded to fp16, its sums are fp32."""
    keys = k.shape[0]
    # keys nobody may see count for nothing, whatever they hold
    k, v = (torch.where(ok.any(0)[:, None], t, torch.zeros_like(t)) for t in (k, v))
    s = q @ k.T / math.sqrt(D)
    s = torch.where(ok, s, torch.full_like(s, -math.inf))
    m = s.amax(1, keepdim=True)
    m = torch.where(m > -math.inf, m, torch.zeros_like(m))
    p = torch.exp(s - m)
    l = p.sum(1, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    out = p @ v
    # a score: 128 products summed in fp32 and scaled (two roundings more), an exponent of that size;
    # numerator and denominator both carry it
    es = 2 * 132 * E32 * (q.abs() @ k.abs().T / math.sqrt(D)).amax(1, keepdim=True)
    rel = es + (keys + 8) * E32  # sums over the keys
    tol = (p @ v.abs()) * (E16 + rel) + out.abs() * E16 + 2.0 ** -24 * (1 + v.abs().amax())
    return out, p, tol, rel


def scores(q, hi, lo, ks):
    """Block scores [M, n_kv, n] fp32 of queries q [M, n_kv, G, D]; hi, lo [n_kv, n, D] codes."""
    a = torch.where(q.double().abs() < math.inf, q.double().abs(), torch.zeros(1).double().to(q.device))
    a = a.amax(-1, keepdim=True)
    r = torch.where(a > 0, 127.0 / a, torch.zeros_like(a)).float()
    c = (q.double() * r.double()).float().round().clamp(-127, 127)
    c = torch.where(q.isnan() | (r == 0), torch.zeros_like(c), c).double()
    sq = (a / torch.full_like(a, 127.0)).float()[..., 0]
    M, n_kv, G, _ = q.shape
    out = torch.empty((M, n_kv, hi.shape[1]), dtype=torch.float32, device=q.device)
    for g in range(n_kv):
        u = (c[:, g].clamp_min(0) @ hi[g].T + c[:, g].clamp_max(0) @ lo[g].T)  # whole numbers
        sc = (u * ks[g].double()).float().double() * sq[:, g, :, None].double()
        out[:, g] = sc.float().amax(1)
    return out


def choose(key, n_first, n_last, k):
    """Indices of the k greatest keys [n] (ties: the lowest index; the first and last ones always),
    ascending."""
    n = len(key)
    held = set(range(min(n_first, n))) | set(range(max(0, n - n_last), n))
    vals = [(-math.inf if x != x else x) for x in key]
    nan = [x != x for x in key]
    for i in sorted(range(n), key=lambda i: (nan[i], -vals[i], i)):
        if len(held) >= k:
            break
        held.add(i)
    return sorted(held)
