"""How products of microscaled matrices are run, on the host: plans within the chip's limits, no candidate that is never taken, and GPU tests that take
every form."""
import os
import random
import subprocess

import pytest

from spoc_b200.build import CSRC, _nvcc
from tests.test_gpu_mx import SHAPES
from tests.test_gpu_mx_forms import FORMS

HERE = os.path.dirname(os.path.abspath(__file__))
SMS = 148


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "mx_plan")
    res = subprocess.run([_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-I", CSRC, "-o", exe, os.path.join(HERE, "mx_plan.cu")],
                         capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stderr

    def run(sizes, sms=SMS):
        text = "\n".join("%d %d %d %d" % s for s in sizes)
        out = subprocess.run([exe, str(sms)], input=text, capture_output=True, text=True, timeout=120, check=True).stdout.splitlines()
        assert len(out) == len(sizes)
        for size, line in zip(sizes, out):
            f = dict(x.split("=") for x in line.split())
            candidates = {tuple(map(int, c.split(":"))) for c in f.pop("candidates").rstrip(",").split(",")}
            yield size, {k: int(v) for k, v in f.items()}, candidates
    return run


def drawn(count, seed=0, most=15):
    rng = random.Random(seed)
    return [(rng.randint(0, 1), *(int(2 ** rng.uniform(0, most)) for _ in range(3))) for _ in range(count)]


@pytest.mark.parametrize("sms", [148, 132, 20])
def test_plans_fit_the_chip(plans, sms):
    for (fp4, m, n, k), p, _ in plans(drawn(20000) + drawn(2000, 1, 27), sms):
        columns = 4 * (2 if fp4 else 1) * (1 + p["groups"])      # of tensor memory a slot of scales
        assert p["stages"] >= 1 and p["slots"] >= 1 and p["slots"] <= p["stages"] <= 12
        assert p["stages"] * p["stage_bytes"] <= 216 * 1024 and p["stage_bytes"] % 1024 == 0
        assert p["tmem_cols"] in (32, 64, 128, 256, 512)
        many = p["splits"] == 1 and p["tiles"] > sms // p["ctas"]
        scales = p["tmem_cols"] - p["slots"] * columns            # where they begin
        assert (p["acc1"] if many else 0) + p["bt"] <= scales and scales % 4 == 0
        assert p["acc1"] >= p["bt"] - 64                          # accumulators overlap by what is drained first
        assert p["bt"] % (8 * p["ctas"]) == 0 and (p["bt"] % 128 == 0 or m <= p["bt"])
        assert p["splits"] <= 8 and (p["splits"] - 1) * p["split_k_blocks"] < p["num_k_blocks"] <= p["splits"] * p["split_k_blocks"]
        assert p["groups"] == -(-p["bt"] // 128)
        if p["splits"] > 1:                                       # partial sums lie in the ring
            assert p["ctas"] == 1 and p["bt"] * 512 <= 216 * 1024


def test_every_candidate_is_taken_by_some_size(plans):
    considered, taken = set(), set()
    for _, p, candidates in plans(drawn(60000)):
        considered |= {(ctas, bt, splits > 1) for ctas, bt, splits in candidates}
        taken.add((p["ctas"], p["bt"], p["splits"] > 1))
    assert taken == considered


def test_the_gpu_tests_take_every_form(plans):
    sizes = [(fp4, *s) for s in SHAPES + FORMS for fp4 in (0, 1)]
    seen = set()
    for (fp4, m, n, k), p, _ in plans(sizes):
        units = SMS // p["ctas"]
        how = "divided" if p["splits"] > 1 else "several" if p["tiles"] > units else "one"
        form = (fp4, p["ctas"], p["bt"], how)
        seen |= {form}
        if p["split_k_blocks"] > p["stages"]:
            seen.add(form[:3] + ("ring turns",))
        if how == "several" and p["tiles"] > 2 * units:
            seen.add((fp4, p["ctas"], "accumulators come round"))
        if p["slots"] < p["stages"]:
            seen.add((fp4, "fewer slots than stages"))
        if how == "several" and p["acc1"] < p["bt"]:
            seen.add((fp4, "accumulators overlap"))
        if p["ctas"] == 2:
            if 0 < n % 256 <= 128:
                seen.add((fp4, p["bt"], "a pair's second block past the last column"))
            if 0 < m % p["bt"] <= p["bt"] // 2:
                seen.add((fp4, p["bt"], "a pair's second block past the last row"))
        if fp4 and p["chunks"] % 2:
            seen.add((p["ctas"], p["bt"], "half a k-block"))
    want = set()
    for fp4 in (0, 1):
        want |= {(fp4, 1, bt, how) for bt in (16, 32, 64, 128) for how in ("one", "divided", "several")}
        want |= {(fp4, 2, bt, how) for bt in (128, 256) for how in ("one", "several", "ring turns")}
        want |= {(fp4, 1, 16, "ring turns"), (fp4, 1, 128, "ring turns"), (fp4, 1, "accumulators come round"), (fp4, 2, "accumulators come round")}
        want |= {(fp4, "fewer slots than stages"), (fp4, "accumulators overlap")}
        want |= {(fp4, bt, f"a pair's second block past the last {what}") for bt in (128, 256) for what in ("column", "row")}
    want |= {(1, bt, "half a k-block") for bt in (16, 64, 128)} | {(2, bt, "half a k-block") for bt in (128, 256)}
    assert want <= seen, sorted(map(str, want - seen))
