"""A plain float64 form of k2b pages and of attention over them, for tests of the decode and prompt kernels.

Tolerance of a kernel's fp16 output against it (`assert_attention`).  The kernels round, relative to the rounded value and by at most
half a step (fp16: u = 2^-11): the low-rank part of a key after each of its rank/16 accumulations, the key after the residual is added,
two products and sums of its rotation, the rotated query (decode) -- at most 6 roundings per key channel; the weight times the value norm
once; the output once.  Roundings of different channels and tokens are independent, so they add in squares: a score
scale * sum_c q_c K_c moves by about scale * |q||K| / sqrt(128) * sqrt(6) * u / sqrt(3), which for the inputs here (|q| = sqrt(128), scale =
1/sqrt(128), |K| <= 8) is 8 / 11.3 * 1.41 * u = u; a weight moves by that much relative, plus u / sqrt(3) for its own rounding.  Output
errors are sums of independently perturbed weights, as the output itself is of the weights: the relative error (2-norm) stays below
sqrt(1 + 1/3 + 1/3) u = 1.3 u = 6.3e-4.  Bound: 1.5e-3 (rows differ in how they concentrate).  A single entry may be five times the
norm-wise bound off, relative to the largest entry of its row.  One token too many or too few among n of like weight moves the output by
about 1 / sqrt(n): 1.5e-2 at 4096, ten times the bound."""

import math

import torch

D = 128
REL = 1.5e-3


def hadamard():
    h = torch.ones(1, 1, dtype=torch.float64)
    for _ in range(7):
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(D)


def pages(K, pool, slots, basis_f16, signs, codebook):
    """Pre-rotation keys and values of page slots, float64 (h_kv, n * 128, 128), from the exported containers."""
    g = pool.geom
    st = {k: v.cpu() for k, v in K.k2b_export_stacks(pool, torch.tensor(slots, dtype=torch.int32, device=pool.pages.device)).items()}
    n, h = len(slots), g.h_kv
    packed = st["res_int_packed"].to(torch.int16)
    code = torch.stack([packed & 15, packed >> 4], -1).reshape(n, h, D, g.page)          # low nibble first
    code = torch.where(code > 7, code - 16, code).double()
    scale = st["res_scale"].double().reshape(n, h, D, g.page // g.group).repeat_interleave(g.group, -1)
    us = st["us"].double().expand(n, h, g.page, g.rank)
    basis = basis_f16.cpu().double().view(h, D, g.rank)
    k = torch.einsum("nhtr,hcr->nhtc", us, basis) + (code * scale).transpose(2, 3)
    idx = torch.stack([(st["v_idx_packed"].long() >> (2 * i)) & 3 for i in range(4)], -1).reshape(n, g.page, h, D)
    v = (codebook.cpu().double()[idx] / math.sqrt(D)) @ hadamard() * signs.cpu().double() * st["v_norm"].double()[..., None]
    return k.permute(1, 0, 2, 3).reshape(h, -1, D), v.permute(2, 0, 1, 3).reshape(h, -1, D)


def rotate(k, cos, sin, pos):
    c, s = cos.cpu().double()[pos], sin.cpu().double()[pos]
    return k * c + torch.cat([-k[..., D // 2:], k[..., : D // 2]], -1) * s


def attend(q, k, v, seen, scale=1.0 / math.sqrt(D)):
    """q (heads, rows, 128), k and v (h_kv, n, 128), seen (rows, n) -> (heads, rows, 128) float64; a row that sees nothing gives 0."""
    h = k.shape[0]
    q = q.cpu().double().reshape(h, -1, q.shape[1], D)
    k = torch.where(seen.any(0)[:, None], k, torch.zeros_like(k))                        # what nobody sees may be anything
    v = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))
    sc = (torch.einsum("hgnd,htd->hgnt", q, k) * scale).masked_fill(~seen, float("-inf"))
    top = sc.amax(-1, keepdim=True) if sc.shape[-1] else torch.full((*sc.shape[:-1], 1), float("-inf"), dtype=torch.float64)
    w = torch.exp(sc - torch.where(top.isinf(), torch.zeros_like(top), top))
    out = torch.einsum("hgnt,htd->hgnd", w, v) / w.sum(-1, keepdim=True).clamp(min=1e-300)
    return out.reshape(-1, q.shape[2], D)


def assert_attention(out, ref, what=""):
    out, ref = out.detach().cpu().double(), ref.double()
    assert torch.isfinite(out).all(), f"{what}: not finite"
    norm = float(ref.norm())
    rel = float((out - ref).norm()) / norm if norm else float(out.abs().max())
    assert rel <= REL, f"{what}: off by {rel:.2e} of the norm"
    worst = ((out - ref).abs().amax(-1) / ref.abs().amax(-1).clamp(min=1e-12))
    worst = float(torch.where(ref.abs().amax(-1) > 0, worst, out.abs().amax(-1)).max())
    assert worst <= 5 * REL, f"{what}: an entry is off by {worst:.2e} of its row's largest"


def fill(K, geom, n_slots, dev, seed):
    """A pool whose slots hold quantized pages of seeded keys and values; returns pool, basis (fp16), signs, codebook."""
    from tests.test_k2b_gpu import make_k2b_inputs

    k, v, basis = make_k2b_inputs(seed, n_slots, geom.h_kv, geom.page, geom.rank, geom.n_coef_heads == geom.h_kv)
    k = k * 4                                                                            # scores with a spread of about 0.5
    pool = K.K2bPool(geom, n_slots, dev)
    signs, cb = K.hadamard_signs(D, 0).to(dev), torch.tensor(K.GAUSSIAN_CODEBOOK[2], device=dev)
    basis = basis.to(dev)
    K.k2b_append(pool, k.to(dev), v.to(dev), basis, signs, cb, torch.arange(n_slots, dtype=torch.int32, device=dev), 1)
    return pool, basis.half().contiguous(), signs, cb


def norms(pool):
    """The fp16 value norms (slots, h_kv, 128) inside the page blocks."""
    return pool.pages[:, :, -256:].view(torch.float16)


def coefs(pool):
    """Coefficients (slots, coef heads, token / 8, rank / 8, token % 8, 8) as they lie in the coefficient blocks of layout 1."""
    g = pool.geom
    return pool.coefs.view(torch.float16).view(pool.n_slots, g.n_coef_heads, 16, g.rank // 8, 8, 8)


def assert_one_step(a, b):
    """Two fp16 outputs of the same float32 values summed in another order: the sums differ by a few float32 roundings (1e-5 of the row's
    largest entry covers 2^7 of them), the rounded values by one fp16 step at most (2^-10 relative) where that crosses a border."""
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    assert ((a - b).abs() <= 2.0 ** -10 * a.abs().maximum(b.abs()) + 1e-5 * a.abs().amax(-1, keepdim=True) + 2.0 ** -24).all()
