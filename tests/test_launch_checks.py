"""What a launch accepts, without a GPU: the runtime's argument checks over
the manifests that the compiler writes."""
import pytest

import group_catalog as cat
import norm_mx_catalog as nc
from hfusion_mi355x import groups as g
from launch_checks import Checked


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return tmp_path_factory.mktemp("checks")


def checked(name, folder, rows=-1):
    return Checked(cat.get(name), folder, options=cat.options(name), rows=rows)


@pytest.mark.parametrize("which", ["norm", "gradient", "codes", "product"])
def test_a_check_costs_little(folder, which):
    """A kernel of a few microseconds waits for its call: the checks of six to
    eight arguments took 1.0 us where their shapes were multiplied and their
    types compared at every launch."""
    name, rows = {"norm": ("ln_rt", 16), "gradient": ("lngrad_wide_rt", 64), "codes": ("quantmx_e2m1_rt", 16),
                  "product": ("linmx_e2m1_rt", 1)}[which]
    c = checked(name, folder, rows)
    assert c.why() == ""
    assert 0 < c.ns() < 250


def test_overlap_of_arguments(folder):
    """A written argument over another is refused, one beside it is not, at
    whatever row count the launch has."""
    for rows in (1, 20, 3000):
        c = checked("lngrad_wide_rt", folder, rows)  # dy x gamma mean rstd dx dgamma dbeta
        assert c.why() == ""
        for out in (5, 6, 7):
            for other in range(8):
                if other == out:
                    continue
                a = c.at[other]
                assert "is written and overlaps" in c.why({out: a})
                assert "is written and overlaps" in c.why({out: a + c.param_bytes(other) - 1})
                assert "is written and overlaps" in c.why({out: a - c.param_bytes(out) + 1})
                assert c.why({out: a + c.param_bytes(other)}) == "" and c.why({out: a - c.param_bytes(out)}) == ""
        # operands may share what they read
        assert c.why({1: c.at[0], 3: c.at[4]}) == ""
    # without rows there is nothing to overlap
    c = checked("lngrad_wide_rt", folder, 0)
    assert c.why({5: c.at[2] + 64}) == "" and "overlaps" in c.why({6: c.at[2]})


@pytest.mark.parametrize("name", ["ln_untied", "lngrad_untied", "quantmx_untied"])
def test_overlap_of_results(folder, name):
    """Results in buffers of their own are destinations too: none over an
    operand, none over another.  (The gradient of few rows reads dy by columns
    while other workgroups write dx.)"""
    c = checked(name, folder)
    n, m = len(c.at), len(c.res)
    assert m > 1 and all(r["tied"] < 0 for r in c.meta["results"]) and c.why() == ""
    for j in range(m):
        for i in range(n):
            assert f"result {j} of" in c.why(res={j: c.at[i]}) and f"overlaps argument {i}" in c.why(res={j: c.at[i]})
            assert "overlaps" in c.why(res={j: c.at[i] + c.param_bytes(i) - 1}) and "overlaps" in c.why(res={j: c.at[i] - c.result_bytes(j) + 1})
            assert c.why(res={j: c.at[i] + c.param_bytes(i)}) == "" and c.why(res={j: c.at[i] - c.result_bytes(j)}) == ""
        for i in range(m):
            if i != j:
                assert "is written and overlaps result" in c.why(res={j: c.res[i]})
                assert c.why(res={j: c.res[i] + c.result_bytes(i)}) == ""
    assert "null device pointer for result 1" in c.why(res={1: 0})


def test_overlap_of_a_result_and_a_written_argument(folder):
    """Some destinations arguments, some not."""
    ir = nc.untied(g.quantize_mx(64, 96)).replace("%x: tensor<64x96xbf16>)", "%x: tensor<64x96xbf16>, %s: tensor<64x3xui8>)") \
        .replace("    %s = tensor.empty() : tensor<64x3xui8>\n", "")
    c = Checked(ir, folder)
    assert [r["tied"] for r in c.meta["results"]] == [-1, 1] and c.why() == ""
    assert "overlaps" in c.why(res={0: c.at[0]}) and "overlaps" in c.why(res={0: c.at[1]}) and "overlaps" in c.why(at={1: c.at[0] + 5})


def test_overlap_of_an_epilogue(folder):
    """A bias is read by every row tile, a factor of a row by every column
    tile: no result over them.  A residual is read where the result is
    written: the two may be one buffer, of elements of one size."""
    for name, rows in (("linmx_e2m1_rt", 65), (nc.linear_name(nc.LINEAR[3]), -1)):
        c = checked(name, folder, rows)  # a w scales bias out
        assert c.why() == ""
        for i in range(4):
            assert f"overlaps argument {i}" in c.why({4: c.at[i]}) and f"overlaps argument {i}" in c.why({4: c.at[i] - 16})
            assert c.why({4: c.at[i] + c.param_bytes(i)}) == ""
    c = checked("linmx_residual", folder)  # a w scales residual factor out
    assert "overlaps argument 4" in c.why({5: c.at[4]}) and "overlaps argument 4" in c.why({5: c.at[4] - 4})
    assert c.why({5: c.at[3]}) == ""
    assert "overlaps argument 3" in c.why({5: c.at[3] + 4}) and "overlaps argument 3" in c.why({5: c.at[3] - 48 * 4})
    c = checked("linmx_residual_bf16", folder)
    assert "overlaps argument 3" in c.why({5: c.at[3]}) and c.why() == ""
    untied = Checked(cat.get("linmx_residual").replace(", %out: tensor<70x48xf32>) ->", ") ->").replace("outs(%out :", "outs(%e5 :"), folder)
    assert [r["tied"] for r in untied.meta["results"]] == [-1]
    assert untied.why() == "" and untied.why(res={0: untied.at[3]}) == "" and "result 0 of" in untied.why(res={0: untied.at[4]})
    assert "overlaps argument 1" in untied.why(res={0: untied.at[1]})


@pytest.mark.parametrize("name", ["ln_rt", "lngrad_rt", "lngrad_plain_rt", "quantmx_e4m3_rt", "dequantmx_e2m1_rt", "linmx_e2m1_rt", "linmx_e4m3_rt"])
def test_tensors_of_no_rows_have_no_address(folder, name):
    """An empty batch: null where a tensor has no rows, and nowhere else."""
    c = checked(name, folder, 0)
    rows = [i for i, p in enumerate(c.meta["params"]) if -1 in p["shape"]]
    null = {i: 0 for i in rows}
    assert rows and c.why(null) == ""
    for i in range(len(c.at)):
        if i not in rows:
            assert c.why({**null, i: 0}) == f"null device pointer for argument {i}"
    c = checked(name, folder, 1)
    for i in rows:
        assert c.why({i: 0}) == f"null device pointer for argument {i}"


def test_where_a_workspace_starts(folder):
    """argmax keeps 64-bit words there, and took any buffer of them; a weight
    as bf16 is read 16 bytes a lane; a group without one takes what comes."""
    for name, rows, on in (("argmax_16", -1, 8), ("lngrad_rt", 9, 16), ("linmx_e2m1_rt", 9, 16), ("ln_rt", 9, 1)):
        c = checked(name, folder, rows)
        for at in range(0x1000, 0x1020):
            assert c.why_workspace(at) == ("" if at % on == 0 else f"a workspace of group @{c.meta['func']} has to start on {on} bytes")
