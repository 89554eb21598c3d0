"""The benchmark's one line on stdout (CPU only)."""

import json

import bench


def test_headline_is_one_short_line(capsys):
    """As many measurements as a run makes: the line stays one that a log's end holds, and nothing is lost."""
    each = {"us": 12345.67, "hbm_frac": 0.1234, "mfma_frac": 0.1234, "max_frac": 0.1234, "samples": 30, "note": "x" * 100}
    line = {"metric": bench.METRIC, "value": 3983.4, "unit": "GB/s", "n_gpus": 1, "steps": 200, "warmup": 20, "ms_per_step": 0.0757,
            "config": {"K": 5120}, "roofline": {"note": "x" * 900}, "floors": each, "workloads": {k: {"a": each, "b": each}
                                                                                                 for k in bench.WORKLOADS},
            "cpu_baseline": each, **{k: {str(i): each for i in range(40)} for k in bench.DETAIL}}
    assert len(json.dumps(line)) > 20000
    bench.emit(line)
    out, err = capsys.readouterr()
    assert out.endswith("\n") and out.count("\n") == 1 and len(out) < 8000
    got = json.loads(out)
    assert {k: line[k] for k in got} == got and not set(got) & set(bench.DETAIL)
    detail = json.loads(err.split("[bench] detail ", 1)[1])
    assert {**got, **detail} == line
