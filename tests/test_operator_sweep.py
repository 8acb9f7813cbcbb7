"""The block operators' arm of the sweeps: its grid and byte counts on the CPU, its rows on a GPU."""
from __future__ import annotations

import json
import math

import pytest

from powermodeling_b200 import sweeps


def test_points_name_every_operator_and_stay_in_memory():
    for quick in (True, False):
        points = sweeps.operator_points(quick)
        assert {p["operator"] for p in points} == {"block_norm", "block_norm_backward", "matvec_w4", "paged_attention"}
        assert len({json.dumps(p, sort_keys=True) for p in points}) == len(points)
        assert all(0 < sweeps.operator_bytes(p) < 6 << 30 for p in points)
    assert len(sweeps.operator_points(True)) < len(sweeps.operator_points(False))


def test_bytes_counted_by_hand():
    assert sweeps.operator_bytes({"operator": "block_norm", "rows": 3, "width": 8}) == 4 * 3 * 8 * 2 + 2 * 8 * 2 + 3 * 8
    assert sweeps.operator_bytes({"operator": "block_norm_backward", "rows": 3, "width": 8}) == 6 * 3 * 8 * 2 + 4 * 8 * 2 + 3 * 8
    # 5 rows of 4 bytes of weights and 2 scales; 2 tokens of 7 values in and 5 out
    assert sweeps.operator_bytes({"operator": "matvec_w4", "tokens": 2, "n": 5, "k": 7, "group_size": 4}) == 5 * (4 + 4) + 2 * 2 * 12
    # 4 old positions and the new one read, the new one written, of 2 x 1 head x 8 values; 2 query heads in and out; 3 pages
    point = {"operator": "paged_attention", "batch": 1, "length": 5, "q_heads": 2, "kv_heads": 1, "head_dim": 8, "page_size": 2}
    assert sweeps.operator_bytes(point) == 2 * 16 * 6 + 2 * 2 * 16 + 4 + 12


def test_sweep_names_its_parts():
    assert "operators" in sweeps.PARTS
    with pytest.raises(SystemExit):
        sweeps.main(["--out", "unused.json", "--only", "operator"])


@pytest.mark.gpu
def test_calls_wait_for_their_operands(monkeypatch):
    import torch
    seen, flags = torch.zeros(1000, device="cuda"), torch.zeros(1000, device="cuda")
    with torch.cuda.stream(torch.cuda.Stream()):          # what a first use waits for is done with
        seen.copy_(flags)
    torch.cuda.synchronize()
    count = iter(range(1000))

    def call(point, seed):
        k = next(count)
        torch.cuda._sleep(50_000_000)                     # some 25 ms before the operand is there
        flags[k:k + 1].fill_(1.0)
        # a call adds what it sees of its operand; nothing is allocated, which would wait
        return lambda: seen[k:k + 1].add_(flags[k:k + 1]).sub_(1.0)
    point = {"operator": "matvec_w4", "tokens": 1, "n": 1 << 16, "k": 1 << 14, "group_size": 128}
    monkeypatch.setattr(sweeps, "operator_points", lambda quick: [point] * 12)        # each on another stream
    monkeypatch.setattr(sweeps, "operator_call", call)
    rows = sweeps.operator_sweep(quick=True)
    assert len(rows) == 12 and not seen.any()


@pytest.mark.gpu
def test_quick_sweep_rows(tmp_path):
    out = tmp_path / "sweep.json"
    assert sweeps.main(["--out", str(out), "--quick", "--only", "operators"]) == 0
    rows = json.loads(out.read_text())["operators"]
    assert [{k: r[k] for k in p} for r, p in zip(rows, sweeps.operator_points(True))] == sweeps.operator_points(True)
    for r in rows:
        assert r["us"] > 0 and math.isfinite(r["us"]) and r["operand_sets"] >= 2
        assert r["gbs"] == pytest.approx(r["bytes"] / r["us"] / 1e3)
        assert r["gbs"] < 20000                           # no call answers without reading its operands


@pytest.mark.gpu
def test_energy_comes_from_windows_that_hold_enough_samples(monkeypatch):
    """A power from two or three samples is no power: the quick sweep has none, a window of a second has one."""
    point = {"operator": "matvec_w4", "tokens": 1, "n": 4096, "k": 4096, "group_size": 128}
    monkeypatch.setattr(sweeps, "operator_points", lambda quick: [point])
    (quick,), (full,) = sweeps.operator_sweep(quick=True), sweeps.operator_sweep(seconds=1.0)
    if "board_power_w" not in full:
        pytest.skip("no power sensor")
    assert quick["board_power_w"] is None and quick["total_pj_per_byte"] is None
    assert full["board_power_w"] > 0
    assert full["total_pj_per_byte"] == pytest.approx(full["board_power_w"] * full["us"] * 1e6 / full["bytes"])
