"""Test infrastructure: the 4-bit group format, cache planes, page tables and attention over a 4-bit cache in plain 64-bit (or host integer) form."""
import torch

PAGE = 64


def encode(x, scale_type=torch.bfloat16):
    """x [..., 32] -> codes (int64) and scales (float64 [...]): d = r(m / -8), c = clamp(floor(x / d + 1/2) + 8, 0, 15)."""
    x = x.double()
    big = x.abs().amax(-1, keepdim=True)
    place = torch.arange(32, device=x.device).expand_as(x)
    first = torch.where(x.abs() == big, place, 99).amin(-1, keepdim=True).clamp(max=31)
    d = (torch.gather(x, -1, first) / -8).to(scale_type).double()
    c = torch.where(d == 0, 8.0, torch.floor(x / torch.where(d == 0, 1.0, d) + 0.5).clamp(-8, 7) + 8)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    c = torch.where(bad, 8.0, c)
    return c.long(), torch.where(bad, float("nan"), d)[..., 0]


def places(d, keys, device):
    """(byte, shift) of every entry [64, D] in a block's codes."""
    p, e = torch.arange(PAGE, device=device)[:, None], torch.arange(d, device=device)[None]
    j, r = e // 32, e % 32
    if keys:
        i = r % 8
        nib = torch.where(i % 2 == 0, i // 2, 4 + i // 2)
        byte = p * (d // 2) + (r // 8) * (d // 8) + j * 4 + nib // 2
        return byte, (4 * (nib % 2)).expand_as(byte)
    n, g, nib = p // 2, r // 4, r % 4
    place = g ^ (2 * (n % 4) if d == 128 else 4 * (n // 2 % 2))
    byte = n * d + place * (d // 8) + j * 4 + 2 * (p % 2) + nib // 2
    return byte, (4 * (nib % 2)).expand_as(byte)


def plane_codes(plane, d, keys):
    """plane [..., block] uint8 -> codes [..., 64, D] and scales [..., 64, D / 32] (float64)."""
    byte, shift = places(d, keys, plane.device)
    c = plane[..., byte.reshape(-1)].long() >> shift.reshape(-1) & 15
    s = plane[..., PAGE * d // 2:].contiguous().view(torch.bfloat16).double()
    return c.unflatten(-1, (PAGE, d)), s.unflatten(-1, (PAGE, d // 32))


def plane_values(plane, d, keys):
    c, s = plane_codes(plane, d, keys)
    return (c - 8).double() * s.repeat_interleave(32, -1)


def make_plane(x, keys):
    """x [pages, heads, 64, D] -> plane bytes that hold it."""
    d = x.shape[-1]
    c, s = encode(x.unflatten(-1, (-1, 32)))
    byte, shift = places(d, keys, x.device)
    codes = torch.zeros(*x.shape[:2], PAGE * d // 2, dtype=torch.int64, device=x.device)
    codes.scatter_add_(-1, byte.reshape(-1).expand(*x.shape[:2], -1), (c.flatten(-2) << shift).flatten(2))
    return torch.cat([codes.to(torch.uint8), s.to(torch.bfloat16).contiguous().view(torch.uint8).flatten(-2)], -1)


def attention(q, k_plane, v_plane, table, kv_lens, rows, scale, window=0, softcap=0.0, sink=None, num_pages=None):
    """q [T, Hq, D] -> float64 (o, sum of p |v| + 2^-24 sum of |v|): rows[b] last positions of each sequence, packed.  (The second is what the result's error
    goes by; its small part stands for weights far below the largest, which fp16 holds to a 2^-35 of that.)"""
    t, hq, d = q.shape
    hkv = k_plane.shape[1]
    num_pages = num_pages or k_plane.shape[0]
    out, mass = (torch.zeros(t, hq, d, dtype=torch.float64, device=q.device) for _ in range(2))
    at = 0
    for b, (n, r) in enumerate(zip(kv_lens, rows)):
        if n > 0 and r > 0:
            ids = table[b, :-(-n // PAGE)].long()
            there = ((ids >= 0) & (ids < num_pages)).repeat_interleave(PAGE)[:n]
            ids = ids.clamp(0, num_pages - 1)
            j, pos = torch.arange(n, device=q.device), torch.arange(n - r, n, device=q.device)[:, None]
            sees = (j <= pos) & there
            if window:
                sees = sees & (j > pos - window)
            for h in range(hkv):
                k = plane_values(k_plane[ids, h], d, True).flatten(0, 1)[:n]
                v = plane_values(v_plane[ids, h], d, False).flatten(0, 1)[:n]
                hs = slice(h * hq // hkv, (h + 1) * hq // hkv)
                x = torch.einsum("ihd,jd->ihj", q[at:at + r, hs].double(), k) * scale
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                x = torch.where(sees[:, None], x, -torch.inf)
                top = x.amax(-1, keepdim=True)
                if sink is not None:
                    top = torch.maximum(top, sink[hs].double()[None, :, None])
                top = torch.where(top == -torch.inf, 0.0, top)
                e = torch.exp(x - top)
                total = e.sum(-1, keepdim=True)
                if sink is not None:
                    total = total + torch.exp(sink[hs].double()[None, :, None] - top)
                p = torch.where(total == 0, 0.0, e / total)
                some = sees.any(0)  # an entry that no row sees has no part in a sum, whatever it is
                v, p = v[some], p[..., some]
                # nor has one that this row does not see
                o = torch.stack([torch.einsum("hj,jd->hd", p[i][:, sees[i, some]], v[sees[i, some]]) for i in range(r)]) if not torch.isfinite(v).all() \
                    else torch.einsum("ihj,jd->ihd", p, v)
                out[at:at + r, hs] = o
                mass[at:at + r, hs] = torch.einsum("ihj,jd->ihd", torch.where(sees[:, None][..., some], p + 2.0 ** -24, p), torch.where(torch.isfinite(v), v.abs(), 0.0))
        at += r
    return out, mass


def page_tables(ctx, new, table, free, num_pages, T):
    """Host lists -> (table, stack, cu, kv, positions, slots), request by request."""
    table, stack = [list(r) for r in table], list(free)
    width, B = len(table[0]), len(ctx)
    for b in range(B):
        if new[b] < 0:
            stack += table[b][:min(-(-max(ctx[b], 0) // PAGE), width)]
    cu, kv, pos, slot, short = [0], [], [0] * T, [-1] * T, False
    for b in range(B):
        c, n = max(ctx[b], 0), max(new[b], 0)
        first, held, after = cu[-1], -(-c // PAGE), -(-(c + n) // PAGE)
        end = first + n
        fits = after <= width and end <= T
        if new[b] < 0:
            kv.append(0)
        else:
            need = after - held if fits else 0
            if need > 0 and (short or need > len(stack)):
                short, fits = True, False
            for i in range(held, held + need if fits else held):
                table[b][i] = stack.pop()
            kv.append(c + n if fits else c)
            for i in range(min(n, max(0, T - first))):
                p = c + i
                pos[first + i] = p
                if fits:
                    page = table[b][p // PAGE]
                    slot[first + i] = page * PAGE + p % PAGE if 0 <= page < num_pages else -1
        cu.append(end)
    return table, stack, [min(x, T) for x in cu], kv, pos, slot


def q4_0_blocks(w):
    """w [N, K] -> (bytes [N, K / 32, 18] of a GGUF file's 4-bit blocks, float64 values)."""
    c, s = encode(w.unflatten(-1, (-1, 32)), torch.float16)
    return blocks_of(c, s), ((c - 8).double() * s[..., None]).flatten(1)


def blocks_of(c, s):
    qs = (c[..., :16] | c[..., 16:] << 4).to(torch.uint8)
    return torch.cat([s.to(torch.float16)[..., None].contiguous().view(torch.uint8), qs], -1).contiguous()
