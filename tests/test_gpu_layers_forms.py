"""The forms of the kernels of layer norm and embedding that other tests' sizes pass by: sums over many rows by every number of threads a row and
piece of a row, both sides of what counts as few rows, and gradients of tables in slices of 1024 columns."""
import pytest
import torch

import test_gpu_embedding as rows_of_a_table
import test_gpu_layer_norm as norm

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32


# threads a row 64 (a wavefront) to 1024; whole pieces, pairs, single elements; more rows than the workgroups take at once
@pytest.mark.parametrize("rows,d", [(5000, 77), (5000, 510), (2600, 1001), (2600, 1002), (2300, 1016), (1500, 1537), (3000, 2048), (1500, 2046),
                                    (700, 4099), (1100, 4094), (1100, 3999), (600, 8191), (700, 8190), (700, 8192), (300, 12288),
                                    (300, 12290), (300, 16383), (700, 16384), (600, 9001)])
@pytest.mark.parametrize("x,w,b,y", [(BF, FP, FP, BF), (FP, FP, BF, FP), (BF, BF, BF, FP), (FP, BF, None, BF)])
def test_sums_over_many_rows(rows, d, x, w, b, y):
    norm.run_and_check(*norm.make(rows, d, x, w, b, y))


# 2^20 elements, and 1024 rows, are still few
@pytest.mark.parametrize("rows,d", [(1024, 1024), (1024, 1025), (1025, 1024), (1023, 1026), (512, 2048), (513, 2048), (256, 4096), (257, 4096),
                                    (64, 16384), (65, 16384), (1024, 64), (1025, 64), (128, 8192), (129, 8192), (1024, 7), (1025, 7)])
@pytest.mark.parametrize("x,y", [(BF, BF), (FP, FP)])
def test_both_sides_of_few_rows(rows, d, x, y):
    norm.run_and_check(*norm.make(rows, d, x, FP, x, y))


@pytest.mark.parametrize("tokens,vocab,d", [(1, 3, 1024), (700, 90, 1024), (3000, 500, 1032), (2000, 3, 4096), (5000, 700, 4096), (900, 40, 2056),
                                            (130, 1, 1536), (1500, 100, 8200), (64, 2, 16384)])
@pytest.mark.parametrize("table,y,scale,padding", [(FP, BF, 1.0, None), (BF, BF, 27.7, 0), (BF, FP, 1.0, -1), (FP, FP, -0.5, None)])
def test_tables_in_slices_of_1024_columns(tokens, vocab, d, table, y, scale, padding):
    ids = rows_of_a_table.zipf(tokens, vocab, seed=tokens)
    rows_of_a_table.run_and_check(ids, *rows_of_a_table.make(ids, vocab, d, table, y), scale, padding)


@pytest.mark.parametrize("form", ["same", "same_but_one", "two_in_turn", "blocks_of_65", "blocks_of_64", "counting"])
@pytest.mark.parametrize("tokens", [63, 64, 65, 129, 4100])
def test_runs_of_equal_tokens_in_wide_tables(tokens, form):
    """Every number of tokens a group of loads ends with (blocks of 1, 2, 3 ... tokens), and runs that end and start inside 64."""
    vocab = 300
    at = torch.arange(tokens, device="cuda")
    ids = {"same": torch.full((tokens,), 33, device="cuda"), "same_but_one": torch.where(at == tokens // 2, 7, 256 + 7),
           "two_in_turn": torch.where(at % 2 == 0, 5, 5 + 256), "blocks_of_65": (at // 65 * 97) % vocab, "blocks_of_64": (at // 64 * 97) % vocab,
           "counting": ((8 * at + 1.0).sqrt() / 2).long() % vocab}[form]
    rows_of_a_table.run_and_check(ids, *rows_of_a_table.make(ids, vocab, 1544, FP, FP))
    rows_of_a_table.run_and_check(ids, *rows_of_a_table.make(ids, vocab, 2048, BF, BF), 2.0, int(ids[0]))
