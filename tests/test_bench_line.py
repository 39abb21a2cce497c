"""CPU: the line that bench.py prints of a whole record."""
import json
import math
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import bench  # noqa: E402

CONTRACT = ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling", "vs_baseline", "dtype", "data", "config")


def record():
    """As long as what is measured: forty configurations and twenty other sizes, each with all it has."""
    third = 100 / 3
    roofline = {"bound": "mfma", "achieved": third, "peak": 157.3, "unit": "TFLOP/s", "frac": third / 157.3}
    cpu = {"value": third, "unit": "TFLOP/s", "cores": 16, "kind": "port", "sample": "s" * 150}
    entry = {"ms": third, "value": third, "unit": "TFLOP/s", "kernel": "mfma_f32_256x128k+strips", "flops_per_launch": 2.0 * 8192 ** 3, "roofline": roofline,
             "cpu_baseline": cpu, "over_batches": {"min": third, "median": third, "max": third}}
    return {"metric": "m" * 70, "value": 147.1334567, "unit": "TFLOP/s", "n_gpus": 1, "steps": 20, "warmup": 5, "ms_per_step": 7.4728912345, "higher_is_better": True,
            "scaling": "weak", "vs_baseline": None, "dtype": "f32", "data": "synthetic", "config": {"workload": "w" * 150, "kernel": "mfma_f32_256x128d"},
            "roofline": dict(roofline, traffic=4822000000, traffic_source="t" * 60, flops_per_launch=2.0 * 8192 ** 3, kernel_ms=third),
            "axpy": {"value": third, "roofline": roofline, "over_batches": entry, "f64_over_batches": entry, "cpu_baseline": cpu,
                     "ceilings": {"copy_GBs": third, "what": "x" * 400}, "placement_GBs": {"f32": {"a": third}}},
            "mlp_step": {"workload": "w" * 150, "ms_per_step": third, "roofline": roofline},
            "configs": {f"3_f32_gemm_configuration_{i}": dict(entry) for i in range(40)},
            "off_benchmark_sizes": {f"f32_gemm_2300x2300x{i}_NN": dict(entry) for i in range(20)},
            "cpu_baseline": cpu, "cpu_baselines": {f"c{i}": cpu for i in range(4)}, "perf_floor": {"ok": True}}


def test_line_is_short_whole_and_true():
    r = record()
    line = bench.one_line(r)
    assert "\n" not in line and len(line) <= bench.LINE_LIMIT
    got = json.loads(line)
    assert set(r) == set(got)
    for key in CONTRACT:
        assert got[key] == r[key] or math.isclose(got[key], r[key], rel_tol=1e-5), key
    assert got["roofline"]["flops_per_launch"] == 2 * 8192 ** 3
    for key in ("configs", "off_benchmark_sizes"):
        assert set(got[key]) == set(r[key])
        for v in got[key].values():
            assert math.isclose(v["value"], 100 / 3, rel_tol=1e-3) and math.isclose(v["frac"], 100 / 3 / 157.3, rel_tol=1e-3) and v["kernel"]


def test_line_without_the_other_workloads():
    r = dict(record(), configs=None, off_benchmark_sizes=None, cpu_baselines=None, mlp_step=None, cpu_baseline=None)
    got = json.loads(bench.one_line(r))
    assert got["configs"] is None and got["cpu_baselines"] is None and got["value"] == 147.133
