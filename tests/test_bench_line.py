"""bench.py's one line of JSON: whole, and short enough to be kept whole by what collects it."""
import json
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import bench  # noqa: E402


def emitted(line, record):
    read, write = os.pipe()
    bench.emit(write, line, str(record))
    os.close(write)
    with os.fdopen(read) as f:
        text = f.read()
    return text, json.loads(record.read_text())


def record():
    with open(os.path.join(ROOT, 'profiles', 'r06', 'k_bench_demux.json')) as f:         # a default run's, 24.5 KB
        return json.load(f)


def test_a_long_line_is_cut_in_extra(tmp_path):
    line = record()
    before = json.dumps(line)
    assert len(before) > bench.MOST_BYTES
    text, whole = emitted(line, tmp_path / 'record')
    got = json.loads(text)
    assert text.count('\n') == 1 and len(text) <= bench.MOST_BYTES
    for key in ('metric', 'value', 'unit', 'n_gpus', 'steps', 'warmup', 'ms_per_step', 'higher_is_better', 'scaling', 'vs_baseline', 'dtype', 'data'):
        assert got[key] == line[key], key                                                 # to the last digit
    for key in ('config', 'roofline', 'cpu_baseline'):
        assert set(got[key]) == set(line[key]) and json.dumps(got[key]).count(':') == json.dumps(line[key]).count(':'), key
    assert got['roofline']['frac'] == pytest.approx(line['roofline']['frac'], rel=1e-5)
    assert got['concordance']['all_fields_bit_exact'] == line['concordance']['all_fields_bit_exact']
    left = set(got['extra']['left_out'])
    assert set(line['extra']) == (set(got['extra']) | left) - {'left_out', 'concordance.unpinned_decision_flips'}
    assert whole == line and json.dumps(line) == before                                    # nothing is lost, the record is as it was


def test_a_short_line_is_whole(tmp_path):
    line = record()
    line['extra'], line['concordance'] = {'ranks': 2}, None
    text, whole = emitted(line, tmp_path / 'record')
    assert json.loads(text)['extra'] == {'ranks': 2} and whole == line and json.loads(text)['value'] == line['value']
