"""The largest plans, without a device: one whose launches would have 2^32 threads
or more is refused when it is set, with FTX_E_RANGE."""
import numpy as np
import pytest

from test_paged_plan import probe, rows  # noqa: F401

KV = 1024


def chains(n, M, npast=0):
    """n sequences of M new tokens after npast shared ones."""
    new, old = (M + 63) // 64, npast // 64
    return [(np.concatenate([np.arange(old), old + i * new + np.arange(new)]), npast, M) for i in range(n)], old + n * new


def refused(seqs, pages, **kw):
    rc, msg, items, _ = probe(seqs, KV, kw.pop("n_head", KV), n_pages=pages, **kw)
    assert rc in (0, -5), msg
    return rc == -5, items


@pytest.mark.parametrize("n,big", [(16383, False), (16384, True)])
def test_workgroups_of_four_waves(n, big):
    """One row tile of 16 rows a sequence and head, 256 threads: 2^24 of them."""
    bad, items = refused(*chains(n, 1))
    assert bad == big
    if not big:
        assert len(items) == n and not items[:, 7].any()


@pytest.mark.parametrize("n,big", [(8191, False), (8192, True)])
@pytest.mark.parametrize("rows", [128], indirect=True)
def test_workgroups_of_eight_waves(n, big, rows):
    """One tile of 128 rows, 512 threads: 2^23 of them."""
    bad, items = refused(*chains(n, 128))
    assert bad == big
    if not big:
        assert len(items) == n and (items[:, 7] == 1).all()


@pytest.mark.parametrize("pages,big", [(8191, False), (8192, True)])
@pytest.mark.parametrize("npast", [0, 64])
def test_new_pages_of_a_store(pages, npast, big):
    """K and V of a page and head a workgroup of 256 threads: 2^24 of them."""
    seqs, total = chains(1, pages * 64, npast)
    assert refused(seqs, total, n_head=0)[0] == big
    # the store of the tokens of many sequences has them along y
    assert not refused(*chains(3, 4096 * 64), n_head=0)[0]


def test_long_contexts_are_not_new_pages():
    """What only attends is bound by its own launches: 2^16 pages seen."""
    seqs, total = chains(1, 1, 64 << 16)
    assert not refused(seqs, total)[0]
    far = np.full((1 << 20) + 1, -1, np.int32)
    far[-3:] = [0, 1, 2]
    rc, msg, _, _ = probe([(far, 64 << 20, 1)], 1, 4, window=100)
    assert rc == 0, msg


def test_given_row_tiles_are_the_threads_own():
    """A test's row tiles reach no plan of another thread."""
    from concurrent.futures import ThreadPoolExecutor

    from xwfes_amd import ftx

    def tiles():
        return set(probe([(np.arange(5), 0, 300)], 2, 8)[2][:, 7])

    force = ftx.load().paged_force_rows
    with ThreadPoolExecutor(1) as other:
        mine = tiles()
        assert mine == {0}
        force(128)
        try:
            assert tiles() == {1} and other.submit(tiles).result() == mine
        finally:
            force(0)
        other.submit(force, 128).result()
        assert tiles() == mine and other.submit(tiles).result() == {1}
