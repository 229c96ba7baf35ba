"""Which kernel, and how many of its workgroups, packed rows over the 4-bit cache are given to. Sums are in another order by another route, so that bits tell them apart."""
import numpy as np
import pytest

from test_kv4_gpu import bits

pytestmark = pytest.mark.gpu


def filled(ctx, pkg, kv, dim, length, page=64, seed=0):
    """A cache of one sequence of `length` positions."""
    rng = np.random.default_rng(dim + length + seed)
    width = -(-length // page)
    pages = pkg.ops.Kv4Pages(ctx, width, page, kv, dim, np.arange(width).reshape(1, width))
    pages.set_lengths([length])
    k, v = (rng.standard_normal((length, kv, dim)).astype(np.float16) for _ in range(2))
    pages.append(k, v, [length])
    return pages, rng


@pytest.mark.parametrize("dim,waves,rows,per_cu", [(256, 4, 1600, 1), (160, 4, 1600, 1), (256, 8, 3200, 1), (128, 4, 3200, 2), (128, 8, 6400, 1), (64, 4, 3200, 2)], ids=str)
def test_no_more_parts_than_run_at_once(ctx, pkg, dim, waves, rows, per_cu):
    """100 query tiles leave room for 2 parts each on 256 CUs that run one workgroup at a time, and for 5 where they run two: more are not made, whatever is asked for."""
    most = 256 * per_cu // 100
    pages, rng = filled(ctx, pkg, 1, dim, rows)
    q = rng.standard_normal((rows, 4, dim)).astype(np.float16)
    got = {}
    for split in (1, 2, 3, 5, 9):
        with ctx.options(HIPC_PROMPT_WAVES=waves, HIPC_PROMPT_SPLIT=split):
            got[split] = bits(pages.prompt_attention(q, [rows]))
    assert not np.array_equal(got[1], got[2])
    for split in (2, 3, 5, 9):
        assert np.array_equal(got[split], got[min(split, most)]), split
    pages.free()


@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("heads,kv,dim,new,behind,many", [(32, 8, 128, 128, 4000, False), (32, 8, 128, 160, 4000, True), (32, 8, 128, 60, 10000, False), (32, 8, 128, 128, 10000, True),
                                                          (32, 8, 128, 60, 30000, False), (32, 8, 128, 96, 30000, True), (4, 1, 256, 256, 200, False), (4, 1, 256, 384, 200, True),
                                                          (4, 1, 256, 384, 10000, True)], ids=str)
def test_a_piece_goes_to_the_kernel_that_its_context_asks_for(ctx, pkg, dtype, heads, kv, dim, new, behind, many):
    """Many rows of one sequence, or few whose keys are many, are those of the kernel for many rows, here with four wavefronts a workgroup; others stay with the kernel for few."""
    pages, rng = filled(ctx, pkg, kv, dim, behind + new)
    q = rng.standard_normal((new, heads, dim)).astype(dtype)
    got = bits(pages.prompt_attention(q, [new]))
    with ctx.options(HIPC_PROMPT_WAVES=4):
        assert np.array_equal(got, bits(pages.prompt_attention(q, [new]))) == many
    pages.free()


@pytest.mark.parametrize("behind,many", [(12000, False), (30000, True)], ids=str)
def test_a_piece_beside_single_tokens_goes_there_later(ctx, pkg, behind, many):
    """100 rows of one sequence and a token of each of five, which hold the same pages: the kernels run in turn, which pays behind 30000 keys and not behind 12000."""
    page, length = 64, behind + 100
    width, rng = -(-length // page), np.random.default_rng(behind)
    pages = pkg.ops.Kv4Pages(ctx, width, page, 8, 128, np.tile(np.arange(width), (6, 1)))
    pages.set_lengths([length] + [behind] * 5)
    k, v = (rng.standard_normal((length, 8, 128)).astype(np.float16) for _ in range(2))
    pages.append(k, v, [length, 0, 0, 0, 0, 0])
    q = rng.standard_normal((105, 32, 128)).astype(np.float16)
    got = bits(pages.prompt_attention(q, [100, 1, 1, 1, 1, 1]))
    with ctx.options(HIPC_PROMPT_WAVES=4):
        forced = bits(pages.prompt_attention(q, [100, 1, 1, 1, 1, 1]))
    assert np.array_equal(got[:100], forced[:100]) == many
    pages.free()
