"""The workspace of vbs_cu_attention_tree on the host: what the query returns
holds every plan up to its description, over sweeps of the sizes that the plan
depends on. Compiled from the library's own source (tests/
tree_plan_harness.cu, PTX only: no GPU, no ptxas)."""
import random
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
PKG = ROOT / "verum-bespoke-singularity_b200"


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("nvcc is not available")
    exe = tmp_path_factory.mktemp("plan") / "tree_plan"
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=compute_100a", "--expt-relaxed-constexpr",
                    "-I", str(PKG / "csrc"), "-I", str(ROOT / "include"), str(ROOT / "tests" / "tree_plan_harness.cu"), "-o", str(exe)],
                   check=True, capture_output=True, timeout=900)

    def run(lines):
        text = "".join(" ".join(str(int(v)) for v in s) + "\n" for s in lines)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True, timeout=600).stdout
        return [[tuple(int(x) for x in item.split(":")) for item in line.split()] for line in out.splitlines()]
    return run


def holds(rows):
    """rows: one description's sweep over ctx_limit, for growing n_tokens."""
    before = None
    for row in rows:
        most = 0
        for i, (plan, ask, *_) in enumerate(row):
            assert plan <= ask and ask % 256 == 0
            assert most <= ask, "shorter contexts asked for more"
            most = ask
            if before is not None:
                assert before[i][1] <= ask, "fewer tokens asked for more"
        before = row


@pytest.mark.parametrize("hd", [32, 64, 80, 128, 200, 256])
@pytest.mark.parametrize("nkh,seqs,group", [(8, 1, 4), (8, 1, 8), (2, 1, 4), (1, 1, 8), (3, 5, 5), (8, 8, 1), (1, 40, 16), (8, 37, 4)])
def test_the_query_holds_every_smaller_plan(plans, hd, nkh, seqs, group):
    tokens = [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 40, 63, 64, 65, 100, 200]
    for clusters in (0, 100, 296):
        for step, limit in ((64, 20000), (4096, 1 << 20)):
            holds(plans([(hd, nkh, seqs, group, n, 0, 0, clusters, step, limit) for n in tokens]))


def test_drawn_descriptions(plans):
    rng = random.Random(7)
    lines = []
    for _ in range(300):
        limit = int(2 ** rng.uniform(6, 28))
        lines.append((rng.choice([8, 64, 96, 128, 136, 256]), rng.choice([1, 2, 3, 8, 40]), int(2 ** rng.uniform(0, 8)),
                      int(2 ** rng.uniform(0, 8)), int(2 ** rng.uniform(0, 12)), rng.choice([0, 0, 1, 1000, 100000]),
                      rng.randrange(2), rng.choice([0, 64, 148, 296]), max(1, limit // 300), limit))
    switched = 0
    for row in plans(lines):
        holds([row])
        switched += len({(rows, joined) for _, _, rows, _, joined in row}) > 1
    assert switched > 30   # the sweeps do cross from one plan to another


@pytest.mark.parametrize("hd,nkh,group,tokens,limit", [(128, 8, 4, 16, 32768), (128, 8, 8, 63, 32768), (64, 2, 4, 7, 32768), (256, 4, 4, 9, 32768),
                                                       (128, 8, 4, 512, 131072), (128, 8, 4, 2048, 131072), (256, 8, 4, 300, 131072)])
def test_the_query_stays_near_what_plans_need(plans, hd, nkh, group, tokens, limit):
    """It is an upper bound, not any: a few times the largest plan of all
    shorter calls, or the sums of all SMs once full of the widest row tiles."""
    counts = sorted(set(range(1, tokens, max(1, tokens // 100))) | {tokens})
    rows = plans([(hd, nkh, 1, group, n, 0, 0, 0, limit // 256, limit) for n in counts])
    assert rows[-1][-1][1] <= max(4 * max(plan for row in rows for plan, *_ in row), 148 * 256 * (8 + 4 * hd) + 512)
