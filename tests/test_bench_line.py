"""The JSON line of bench.py: whoever keeps the last 8 KB of its output reads all of it."""
import glob
import json
import math
import os

import pytest

from tools import bench_parts

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CONTRACT = ('metric', 'value', 'unit', 'n_gpus', 'steps', 'warmup', 'ms_per_step', 'higher_is_better', 'scaling', 'vs_baseline', 'dtype', 'data')
FILES = [f for f in sorted(glob.glob(os.path.join(ROOT, 'profiles', 'r0[3-6]_bench_*.json'))) if os.path.getsize(f) > 2000]


@pytest.mark.parametrize('path', FILES, ids=os.path.basename)
def test_a_measured_line_is_short_and_keeps_what_counts(path):
    out = json.load(open(path))
    line = bench_parts.brief_line(out)
    assert len(line) <= bench_parts.LINE_LIMIT and '\n' not in line
    got = json.loads(line)
    if len(json.dumps(out)) <= bench_parts.LINE_LIMIT:
        assert got == out
        return
    for k in CONTRACT:
        assert got[k] == out[k], k
    for part in ('config', 'roofline'):
        for k, v in out[part].items():
            if isinstance(v, (int, float)) and not isinstance(v, bool) and math.isfinite(v):
                assert abs(got[part][k] - v) <= 1e-5 * abs(v), (part, k)
            elif not isinstance(v, (dict, list, str)) or (isinstance(v, str) and len(v) <= 60):
                assert got[part][k] == v, (part, k)
    assert got['left_out'] and not any(n in CONTRACT for n in got['left_out'])


def test_short_and_odd_lines():
    assert bench_parts.brief_line({'a': 1.23456789012}) == '{"a": 1.23456789012}'
    out = {'value': 1.23456789012, 'config': {'note': 'x' * 300, 'model': 'm', 'n': 3, 'nan': math.nan, 'list': list(range(3000))}, 'roofline': {'frac': 0.123456789, 'deep': {'a': ['y' * 50] * 400}},
           'extra': {str(k): 0.1234567890123 for k in range(500)}, 'small': {'a': 1}}
    got = json.loads(bench_parts.brief_line(out))
    assert got['value'] == 1.23456789012 and got['config']['model'] == 'm' and math.isnan(got['config']['nan']) and got['roofline'] == {'frac': 0.123457} and got['small'] == {'a': 1}
    assert got['left_out'] == ['long texts', 'roofline.deep', 'config.list', 'extra'] and len(json.dumps(got)) <= bench_parts.LINE_LIMIT
    assert len(out['config']['list']) == 3000                               # what was given stays as it was
