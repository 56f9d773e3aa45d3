"""CPU: the line that bench.py prints stays short enough to be kept whole at the end of a log."""
import json
import os

import bench

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_line_of_a_full_run_is_short():
    """A recorded run of every leg (22.9 kB when its line held all of them): the headline's fields stay as they are, the others keep their numbers."""
    with open(os.path.join(ROOT, "profiles", "r06_final_bench.json")) as f:
        full = json.loads([line for line in f if line.startswith('{"metric"')][0])
    assert len(json.dumps(full)) > 20000
    line = bench.bench_line(full)
    text = json.dumps(line)
    assert len(text) < 10000 and json.loads(text) == line and "\n" not in text
    assert list(line) == list(full)
    for key in ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling", "vs_baseline", "dtype", "data", "config", "roofline",
                "cpu_baseline", "parity_check", "passages_per_s", "uncertified_queries"):
        assert line[key] == full[key], key
    for key in ("config5", "real_size", "splade_search", "e5_large_encode"):
        numbers = {k: v for k, v in full[key].items() if isinstance(v, (int, float))}
        assert numbers and all(line[key][k] == v for k, v in numbers.items()), key
    assert line["larger_k"] == len(full["larger_k"])
