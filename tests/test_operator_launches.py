"""The operators' launches at sizes that no test could run, and those that the GPU tests of single
paths rely on: the library's host code on the host model of the HIP runtime (``csrc/host_check``),
which takes what HIP takes, at least one thread and less than 2^32 of them in a dimension."""

from __future__ import annotations

import pytest

import test_operators_sizes_gpu as sizes
from test_host_sanitize import _run, driver  # noqa: F401  (a fixture)

F32, BF16 = 0, 1
E_ARG = -4


def _launches(driver, *cases):  # noqa: F811
    """For each case, its return code, its scratch and its launches: [(kernel, blocks, threads)]."""
    out, now = [], []
    for line in _run(driver, "launches", *cases).splitlines():
        if line.startswith("= "):
            _, _, rc, work = line.split()
            out.append((int(rc), int(work), now))
            now = []
        else:
            x, y, threads, name = line.split(" ", 3)
            name = name.removeprefix("void ").split("(")[0].replace("pots::", "")
            now.append((name, int(x) * int(y), int(threads)))
    assert len(out) == len(cases)
    return out


@pytest.mark.parametrize("case", [
    f"embedding_forward,{1 << 24},1024,1000,{F32}",    # 2^32 chunks of 16 bytes
    f"embedding_forward,{1 << 24},1048576,1000,{F32}",
])
def test_looked_up_rows_past_a_launch(driver, case):  # noqa: F811
    (rc, _, launches), = _launches(driver, case)
    assert rc == 0
    tokens, dim = (int(x) for x in case.split(",")[1:3])
    threads = sum(x * t for _, x, t in launches)
    assert threads >= tokens * dim // 4 and all(n == "embed_rows<Fp32>" for n, _, _ in launches)


@pytest.mark.parametrize("tokens", [0, 1, 200, 257, 40000])
@pytest.mark.parametrize("vocab", [(1 << 28) + 5, 1 << 30])
def test_dense_gradients_of_tables_past_a_launch(driver, tokens, vocab):  # noqa: F811
    """A block of zeros for every 16 rows of the table would be 2^32 threads."""
    (rc, _, launches), = _launches(driver, f"embedding_backward,{tokens},8,{vocab},{BF16},0")
    assert rc == 0 and "embed_sum" in " ".join(n for n, _, _ in launches)


@pytest.mark.parametrize("rows, vocab", [(1 << 20, 1 << 20), (1 << 24, 40000), (1 << 22, 1 << 18),
                                         (129, 1 << 24), (5, 1 << 24)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_losses_of_more_tiles_than_a_launch(driver, rows, vocab, dtype):  # noqa: F811
    """2^23 tiles of 512 threads and more: the vocabulary is taken in pieces. Every row meets every
    vocabulary entry once."""
    (rc, _, launches), = _launches(driver, f"vocab_loss_forward,{rows},64,{vocab},{dtype}")
    assert rc == 0
    area = {"256u, 256u": 1 << 16, "128u, 128u": 1 << 14, "256u, 32u": 1 << 13,
            "128u, 64u": 1 << 13}
    done = sum(x * next(v for k, v in area.items() if k in n)
               for n, x, _ in launches if n.startswith("loss_scores"))
    assert rows * vocab <= done <= 1.25 * (rows + 255) * (vocab + 255)


@pytest.mark.parametrize("rows, vocab", [(1 << 24, 100), (1 << 20, 1 << 16), (1, 1 << 24)])
def test_gradients_of_as_many_rows_as_the_loss_takes(driver, rows, vocab):  # noqa: F811
    (rc, _, launches), = _launches(driver, f"vocab_loss_backward,{rows},64,{vocab},{BF16}")
    assert rc == 0 and launches[-1][0] == "loss_join<Bf16>"


@pytest.mark.parametrize("case, most", [
    (f"attention_forward,{1 << 20},1,1,{{}},8,{BF16}", 15 * 128),
    (f"attention_backward,{1 << 20},1,1,{{}},8,{BF16}", 15 * 128),
    (f"attention_forward,1,{1 << 20},{1 << 20},{{}},128,{F32}", 15 * 128),
    (f"attention_backward,1,{1 << 20},{1 << 20},{{}},128,{F32}", 7 * 128)])
def test_attention_of_more_rows_than_a_launch(driver, case, most):  # noqa: F811
    """Below 2^24 blocks of 128 rows; from there on the sizes are out of range, and nothing is
    enqueued."""
    good, bad = _launches(driver, case.format(most), case.format(most + 1))
    assert good[0] == 0 and good[2]
    assert bad[0] == E_ARG and not bad[2]


@pytest.mark.parametrize("case", sizes.LOSSES)
def test_what_the_sizes_of_the_loss_reach(driver, case):  # noqa: F811
    dtype, rows, d, vocab, scores, dx, dw, forward, backward = case
    what = f"{rows},{d},{vocab},{BF16 if dtype == sizes.BF else F32}"
    a, b = (x[2] for x in _launches(driver, f"vocab_loss_forward,{what}",
                                    f"vocab_loss_backward,{what}"))
    tiles = [n for n, _, _ in a if n.startswith("loss_scores")]
    assert len(tiles) == forward and all(f"Tile<false, false, {scores}" in n for n in tiles)
    tiles = [n for n, _, _ in b if n.startswith("loss_products")]
    assert len(tiles) == backward
    assert all(f"Tile<true, false, {dx}" in n and f"Tile<true, true, {dw}" in n for n in tiles)


def test_the_sizes_of_the_loss_reach_every_tile():
    assert {c[4] for c in sizes.LOSSES} == {sizes.DIRECT, sizes.NARROW_DIRECT, sizes.LARGE,
                                            sizes.MEDIUM, sizes.NARROW}
    assert {c[5] for c in sizes.LOSSES} == {sizes.LARGE, sizes.TRIMMED, sizes.MEDIUM,
                                            sizes.NARROW_X}
    for tile in (sizes.LARGE, sizes.TRIMMED):  # those of whole batches, in both types
        assert {c[0] for c in sizes.LOSSES if c[5] == tile} == {sizes.BF, sizes.F32}


@pytest.mark.parametrize("tokens, d, vocab", sizes.TABLES)
def test_what_the_sizes_of_the_tables_reach(driver, tokens, d, vocab):  # noqa: F811
    (_, _, launches), = _launches(driver, f"embedding_backward,{tokens},{d},{vocab},{F32},0")
    assert vocab * d * 4 > 256 << 20
    by = {n.split("<")[0]: x for n, x, _ in launches}
    # blocks beyond those of the tokens, 32 to one that orders: zeros are written there
    assert by["embed_order"] > -(-tokens // 32) and "embed_join" in by
    assert ("embed_merge" in by) == (tokens > 16384)
