"""The result line of bench.py (no GPU): whole in its top-level keys, short enough for a log's tail."""
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_result_line_is_short_and_keeps_the_headline():
    if ROOT not in sys.path:
        sys.path.insert(0, ROOT)
    import bench
    nested = {f"workload_{i}": {"bound": "hbm", "achieved": 1.0, "kernel": "k" * 40, "traffic": None} for i in range(60)}
    record = {"metric": "m", "value": 1.0, "unit": "us", "n_gpus": 1, "config": {"M": 1}, "roofline": {"frac": 0.8, "nested": {"frac": 0.4}},
              "cpu_baseline": {"value": 2.0, "unit": "us", "leg": {"value": 3.0}},
              "extra": {"gemv_us": 5.0, "flash_attn_e5m2_h1_d64_L128_us": 6.0, "roofline": nested, "roofline_mfma": nested}}
    line = bench.result_line(record)
    assert list(line) == list(record) and line["roofline"] == record["roofline"] and line["config"] == record["config"]
    assert line["cpu_baseline"] == {"value": 2.0, "unit": "us"} and line["extra"] == {"gemv_us": 5.0}
    assert record["extra"]["roofline"] is nested and "leg" in record["cpu_baseline"]       # the whole record stays as it was
    assert len(json.dumps(line)) < 1000
    assert bench.result_line(dict(record, cpu_baseline=None))["cpu_baseline"] is None      # --no-cpu
