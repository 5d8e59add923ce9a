"""The log decays that linear attention's passes read (chainer_amd/csrc/attend_decay_row.h), on the CPU: a segment of a sequence's last row alone has no row behind it to read."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which('g++') is None, reason='g++ not available')
def test_decays_are_read_inside_the_sequence(tmp_path):
    exe = str(tmp_path / 'attend_decay_row_test')
    subprocess.run(['g++', '-std=c++17', '-O1', '-Wall', '-Werror', '-I', os.path.join(ROOT, 'chainer_amd', 'csrc'), os.path.join(ROOT, 'tests', 'cpp', 'attend_decay_row_test.cc'), '-o', exe],
                   check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and 'all checks passed' in r.stdout, r.stdout + r.stderr


def test_both_kernels_read_decays_by_that_rule():
    for name in ('linear_attention.hip', 'linear_attention_half.hip'):
        with open(os.path.join(ROOT, 'chainer_amd', 'csrc', name)) as f:
            source = f.read()
        assert source.count('gp[') == source.count('gp[AttendDecayRow(') == 1, name
