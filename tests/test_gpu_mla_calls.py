"""GPU: calls of the absorbed attention that its description allows and that
lie outside the sizes of a decode step: chunks of a prompt, thousands of
sequences, the largest number of heads, short tree masks and pages that
sequences share; against tests/mla_ref.py."""
import numpy as np
import pytest

import mla_ref as R
from test_gpu_mla import Paged, check_attend, dev, fill, m, pack_tree, run_attend  # noqa: F401  (m: the context fixture)

pytestmark = pytest.mark.gpu


def chain(lens):
    return [np.tril(np.ones((n, n), bool)) for _, n in lens]


@pytest.mark.parametrize("fmt", R.FORMATS)
@pytest.mark.parametrize("lens,heads,latent", [([(0, 400)], 16, 512), ([(300, 257), (0, 320)], 8, 128), ([(70, 520)], 3, 256)])
def test_prompt_chunks(m, cuda_lib, fmt, lens, heads, latent):  # noqa: F811
    """Causal chunks of several hundred tokens, on an empty context and behind rows."""
    g = Paged(cuda_lib, lens, fmt, latent, 64, seed=7)
    fill(g, 7)
    q = np.random.default_rng(7).standard_normal((g.T, heads, latent + 64))
    scale = 1.5 / np.sqrt(latent + 64)
    out, lse = run_attend(m, g, q, scale, R.kind(fmt))
    check_attend(g, q, scale, out, lse, chain(lens))


@pytest.mark.parametrize("fmt", [R.BF16, R.FP8_F16])
def test_most_sequences(m, cuda_lib, fmt):  # noqa: F811
    """4096 sequences, some of them empty, of one to three tokens."""
    lens = [((b * 7) % 90, (b * 5) % 4) for b in range(4096)]
    g = Paged(cuda_lib, lens, fmt, 128, 16, seed=8)
    fill(g, 8)
    q = np.random.default_rng(8).standard_normal((g.T, 2, 192))
    out, lse = run_attend(m, g, q, 0.1, R.kind(fmt))
    check_attend(g, q, 0.1, out, lse, chain(lens))


@pytest.mark.parametrize("fmt", [R.F16, R.FP8_BF16])
def test_most_heads(m, cuda_lib, fmt):  # noqa: F811
    lens = [(130, 2), (5, 1)]
    g = Paged(cuda_lib, lens, fmt, 128, 64, seed=9)
    fill(g, 9)
    q = np.random.default_rng(9).standard_normal((g.T, 1024, 192))
    out, lse = run_attend(m, g, q, 0.1, R.kind(fmt))
    check_attend(g, q, 0.1, out, lse, chain(lens))


@pytest.mark.parametrize("fmt", [R.BF16, R.FP8_F16])
@pytest.mark.parametrize("ctx", [0, 45, 64])
def test_tree_words_that_end_before_the_rows(m, cuda_lib, fmt, ctx):  # noqa: F811
    """Rows of the call that tree_words does not reach are not seen, not even by their own token."""
    n = 70
    g = Paged(cuda_lib, [(ctx, n)], fmt, 128, 16, seed=10)
    fill(g, 10)
    sees = np.tril(np.ones((n, n), bool))
    short = sees.copy()
    short[:, 32:] = False
    q = np.random.default_rng(10).standard_normal((n, 5, 192))
    out, lse = run_attend(m, g, q, 0.1, R.kind(fmt), tree=pack_tree(sees[:, :32], 1))
    check_attend(g, q, 0.1, out, lse, [short])


@pytest.mark.parametrize("fmt", [R.F16, R.FP8_BF16])
def test_pages_that_sequences_share(m, cuda_lib, fmt):  # noqa: F811
    """Two sequences whose first pages are the same (a common prefix), and one that lists a page twice."""
    lens = [(150, 2), (150, 1), (90, 3)]
    g = Paged(cuda_lib, lens, fmt, 256, 32, seed=11)
    g.table[1, :4] = g.table[0, :4]
    g.table[2, 1] = g.table[2, 0]
    g.bufs[2] = dev(g.table)
    fill(g, 11)
    q = np.random.default_rng(11).standard_normal((g.T, 20, 320))
    out, lse = run_attend(m, g, q, 0.1, R.kind(fmt))
    check_attend(g, q, 0.1, out, lse, chain(lens))


def test_output_in_the_querys_place_is_refused(m, cuda_lib):  # noqa: F811
    import torch
    F = cuda_lib
    g = Paged(F, [(8, 1)], R.BF16, 128, 8)
    ws = torch.empty(m.mla_workspace_bytes(128), dtype=torch.uint8, device="cuda")
    a, b = (torch.zeros(1, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    before = m.kernel_launches
    for q_latent, q_rope in ((a, b), (b, a)):
        with pytest.raises(F.MoeError, match="same buffer"):
            m.mla_attention_device(g.kv, g.batch(), q_latent, (256, 128), q_rope, (256, 128), 2, 0.1, a, (256, 128), ws, ws.numel())
    assert m.kernel_launches == before


@pytest.mark.parametrize("fmt", R.FORMATS)
def test_lse_of_a_few_equal_scores(m, cuda_lib, fmt):  # noqa: F811
    """Scores of zero over 1 to 300 rows: lse = log n, within a step or two of fp32 (log2 of n: 1 ulp, one addition, one
    product by a rounded ln 2; absolute 2^-22 where the reference's own size cancels)."""
    lens = [(0, 1), (1, 1), (2, 1), (63, 1), (299, 1)]
    g = Paged(cuda_lib, lens, fmt, 128, 16, seed=12)
    fill(g, 12)
    out, lse = run_attend(m, g, np.zeros((g.T, 3, 192)), 0.5, R.kind(fmt))
    want = np.log([c + n for c, n in lens])[:, None]
    assert np.all(np.abs(lse - want) <= 2.0 ** -22 * (1 + want)), lse - want
    check_attend(g, np.zeros((g.T, 3, 192)), 0.5, out, lse, chain(lens))
