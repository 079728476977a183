"""bench.py where the reference's library cannot be built: its reference arm says so, and the other arm's lines beside
it do, in place of ending the run."""
import json
import subprocess
import sys

import pytest

pytest.importorskip("torch")


@pytest.fixture
def bench(repo, monkeypatch, tmp_path):
    monkeypatch.syspath_prepend(str(repo))
    import bench as b
    import oracle_bind
    monkeypatch.setattr(oracle_bind, "REF_SO", tmp_path / "absent.so")
    return b


def test_the_reference_arm_is_unavailable(bench, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["bench.py", "--impl", "reference", "--steps", "1"])
    assert bench.main() == 0
    line = json.loads(capsys.readouterr().out.strip())
    assert line["impl"] == "reference" and line["unavailable"] and "\n" not in line["unavailable"] and "value" not in line


def test_the_reference_arm_as_a_process(repo):
    from oracle_bind import REF_SO
    if REF_SO.exists():
        pytest.skip("the reference's library is here")
    r = subprocess.run([sys.executable, str(repo / "bench.py"), "--impl", "reference", "--steps", "1"], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-500:]
    assert json.loads(r.stdout)["unavailable"]


def test_the_single_expert_lines_go_without_it(bench, monkeypatch):
    class Op:
        def __init__(self, *a, **k):
            pass

        def run(self, i, s):
            pass

        def bytes_per_call(self):
            return 529408

    import exl3b200.layer as layer
    monkeypatch.setattr(layer, "Linears", Op)
    monkeypatch.setattr(layer, "ExpertMlps", Op)
    monkeypatch.setattr(bench, "_graph_time", lambda run_all, reps=5: 1000.0)
    res = bench.single_expert_configs(None, 6500.0, with_cpu=True)
    lines = [res["config1_linear_16x2048_to_512"], *res["config2_expert_mlp_2048x512_K4"].values()]
    assert len(lines) == 5
    for line in lines:
        assert line["us"] > 0 and line["cpu_reference"]["unavailable"] and "speedup_vs_cpu" not in line
