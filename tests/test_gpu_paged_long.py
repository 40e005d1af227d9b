"""Attention over pages in pieces whose K passes 2^32 bytes, on the GPU: a table that names one page again and again, so that
the pool stays small and the result is known in closed form."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mako_attn as M  # noqa: E402
import pages_ref as R  # noqa: E402
from test_gpu_paged import gen, ints, space  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,few,many", [(64, 1, 129), (128, 1, 129), (256, 1, 65)])
@pytest.mark.parametrize("form", ["few", "many"])
def test_a_piece_past_32_bits(dim, few, many, form, dtype):
    """One sequence of 2^32 bytes of K and some keys more. With more column blocks (an odd group: one a head) than half the CUs
    there is one range, so every workgroup's piece is the whole sequence.

    Bounds, relative to sum w |v|: the probabilities' rounding; the running sums in 32 bits, a rounding 2^-24 each for every four
    keys of the products with v (an instruction adds 16) and every tile of the weights' sum; the scores' errors (pages_ref). Of
    the log-sums: the latter two. Were tiles past 2^32 bytes read as zeros, they would weigh exp(0) where rows have exp(4)."""
    n = few if form == "few" else many
    page, g = 4096, gen(dim + n)
    heads = torch.cuda.get_device_properties(0).multi_processor_count // 2 + 1
    heads += heads % 2 == 0
    keys = (1 << 32) // (2 * dim) + 3 * 64 + 17
    ctx, max_pages = keys - n, -(-keys // page)
    q, k, v = (torch.randn((h, m, dim), generator=g, device="cuda") * 0.5 for h, m in ((heads, n), (1, page), (1, page)))
    q[..., 0], k[..., 0], v = 4.0, math.sqrt(dim), v * 0.25 + 1  # scores of 4 and more or less
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    table = torch.zeros((1, max_pages), dtype=torch.int32, device="cuda")
    a = M.paged_args(batch=1, rows=n, heads=heads, kv_heads=1, dim=dim, pages=1, page=page, max_pages=max_pages, max_new=n,
                     max_ctx=keys)
    o = torch.zeros((n, heads * dim), device="cuda")
    lse = torch.zeros((heads, n), device="cuda")
    M.attn_paged(a, q, k[None], v[None], table, ints([ctx]), o, space(M.attn_paged_workspace(a)), starts=ints([0, n]), lse=lse)
    torch.cuda.synchronize()

    seen = ctx + 1 + torch.arange(n, device="cuda")
    count = (seen // page)[:, None] + (torch.arange(page, device="cuda") < (seen % page)[:, None])  # of the page's rows
    kk, vv = k[0].double(), v[0].double()
    got = o.view(n, heads, dim).double()
    for h in range(heads):
        s = torch.matmul(q[h].double(), kk.t().contiguous()) * a.scale + count.double().log()
        w = torch.softmax(s, 1)
        want, size = torch.matmul(w, vv), torch.matmul(w, vv.abs())
        most = float((torch.matmul(q[h].double().abs(), kk.abs().t().contiguous()) * a.scale).amax())
        ds = 2.0 ** -24 * ((dim + 2) * most + most + 8)
        sums = keys / 64 * 2.0 ** -24
        tol = size * (R.half_step(dtype) + keys / 4 * 2.0 ** -24 + sums + 2.5 * ds) * 1.01 + 1e-6
        assert ((got[:, h] - want).abs() <= tol).all(), (h, float((got[:, h] - want).abs().amax()))
        off = (lse[h].double() - torch.logsumexp(s, 1)).abs()
        assert (off <= (sums + 64 * 2.0 ** -24 + ds) * 1.01 + 2.0 ** -22 * 32).all(), (h, float(off.amax()))
