"""The vocabulary projection's operators, written from their definitions in 64
bits (include/pesti_sampler.h): the checker of their tests.  Tensors stay on
the device they come on."""
import torch


def cross_entropy(hidden, head, target, weight=None, eps=0.0, zeta=0.0, up=None):
    """dict of loss [N], lse [N], z's largest sum of magnitudes per row, the
    gradients of sum(up * loss) for hidden and head, |G|, and both gradients'
    sums of magnitudes, in which tolerances are counted."""
    h, w = hidden.detach().double(), head.detach().double()
    (N, D), V = h.shape, w.shape[0]
    t = target.long()
    live = (t >= 0) & (t < V)
    a = torch.ones(N, dtype=torch.float64, device=h.device) if weight is None else weight.detach().double()
    live = live & (a != 0)
    at = torch.where(live, t, torch.zeros_like(t))
    h = torch.where(live[:, None], h, torch.zeros_like(h))
    z = h @ w.T
    size = h.abs() @ w.abs().T
    m = z.amax(1, keepdim=True)
    lse = (m + (z - m).exp().sum(1, keepdim=True).log()).squeeze(1)
    chosen = z.gather(1, at[:, None]).squeeze(1)
    loss = a * (lse - (1 - eps) * chosen - eps * z.mean(1) + zeta * lse ** 2)
    a = torch.where(live, a if up is None else a * up.detach().double(), torch.zeros_like(a))
    p = (z - lse[:, None]).exp() * (1 + 2 * zeta * lse)[:, None]
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1 - eps)
    G = torch.where(live[:, None], (p - hot - eps / V) * a[:, None], torch.zeros_like(p))
    # what is added up to G, without cancellation
    parts = torch.where(live[:, None], (p.abs() + hot + eps / V) * a.abs()[:, None], torch.zeros_like(p))
    zero = torch.zeros_like(lse)
    return {"live": live, "loss": torch.where(live, loss, zero), "lse": torch.where(live, lse, zero),
            "size": torch.where(live, size.amax(1), zero), "G": G, "parts": parts,
            "p": torch.where(live[:, None], p.abs() * a.abs()[:, None], torch.zeros_like(p)),
            "grad_hidden": G @ w, "grad_head": G.T @ h, "abs_head": w.abs(), "abs_hidden": h.abs()}


def quantize(head, group):
    """(q [V, D] whole numbers, scale [V, ceil(D / group)] bfloat16) of finite weights."""
    V, D = head.shape
    n = -(-D // group)
    w = torch.zeros(V, n * group, dtype=torch.float64, device=head.device)
    w[:, :D] = head.double()
    w = w.view(V, n, group)
    order = torch.arange(group, device=w.device).expand_as(w)
    size = w.abs()
    first = torch.where(size == size.amax(2, keepdim=True), order, torch.full_like(order, group)).amin(2, keepdim=True)
    m = w.gather(2, first)
    scale = (m / -8).float().to(torch.bfloat16)  # f32 values: the division is exact above subnormals
    s = scale.double()
    q = torch.round(w / torch.where(s == 0, torch.ones_like(s), s))  # halves to even
    q = torch.where(s == 0, torch.zeros_like(q), q.clamp(-8, 7))
    return q.reshape(V, -1)[:, :D], scale.squeeze(2)


def held_values(q, scale, group):
    """The weight that q and scale stand for, in 64 bits."""
    return q.double() * scale.double().repeat_interleave(group, 1)[:, :q.shape[1]]


def unpack(packed, V, D):
    """q [V, D] from the library's layout, tiles of 64 rows and 128 columns: word j
    of chunk t ^ (row // 2 % 4) of a row holds the tile's columns 32j + 8t to
    32j + 8t + 7, the first lowest."""
    T, B = packed.shape[:2]
    b = packed.cpu().view(T, B, 64, 4, 4, 4).long()          # tile, block, row, chunk, j, byte
    nib = torch.stack([b & 15, b >> 4], -1).reshape(T, B, 64, 4, 4, 8)
    row, t = torch.arange(64)[:, None], torch.arange(4)[None, :]
    nib = nib[:, :, row, t ^ (row // 2 % 4)]                  # tile, block, row, t, j, column
    q = nib.permute(0, 2, 1, 4, 3, 5).reshape(T * 64, B * 128)
    return (q[:V, :D] - 8).to(packed.device)
