"""Plans of programs with int4_matmul and the workspace that they take, without a GPU: allocation-free executions have 64 MiB
for all temporaries of a program."""
import pytest

from ryft_amd import operators, pjrt

SCRATCH = 64 << 20


def planned(client, module):
    exe = client.compile(pjrt.Program.mlir(module))
    return exe.describe_plan(), exe.executable().memory_statistics()["temp_size_in_bytes"]


def products(text):
    """Each int4_matmul's line, without its number."""
    return [ln.split(": ", 1)[1] for ln in text.split("\n") if ": int4_matmul " in ln]


# ------------------------------------------------------------------------------------------------ one product
@pytest.mark.parametrize("rows, inner, group", [(17, 1 << 22, 32), (17, 1 << 22, 128), (300, 1 << 20, 128), (2048, 1 << 21, 64)])
def test_rows_too_long_for_tiles_go_without_a_workspace(compile_client, rows, inner, group):
    text, temp = planned(compile_client, operators.int4_matmul_module(rows=rows, inner=inner, columns=64, group=group))
    assert " few" in text and temp == 0


@pytest.mark.parametrize("rows, inner, columns, group", [(17, 1 << 18, 64, 128), (512, 25600, 4096, 32), (1024, 52352, 4096, 128),
                                                         (40, 1 << 19, 300, 32), (100_000, 64, 4096, 32)])
def test_one_product_fits_the_scratch(compile_client, rows, inner, columns, group):
    text, temp = planned(compile_client, operators.int4_matmul_module(rows=rows, inner=inner, columns=columns, group=group))
    assert " tile=" in text and 0 < temp <= SCRATCH
