"""Calls past the limits of a launch are refused on the host, before any HIP call."""
import pytest

from test_q4_host import GOOD, ROPE, _abort_run


@pytest.mark.parametrize("n,rows,off", [(1, 1 << 24, 16), (65535, 13 << 20, 16), (65535, 65535 * 210, None)])
def test_rotation_and_append_of_more_threads_than_a_launch_has(n, rows, off):
    """18 workgroups of 256 threads a page (14B): 2^32 threads and more"""
    call = ROPE.format(**{**GOOD, "n": n, "rows": rows, "off": off})
    r = _abort_run(f"import nova_amd; n = nova_amd.load('qwen25_14b'); {call}")
    assert r.returncode == -6 and "requirement failed: wgs * QT <= UINT32_MAX" in r.stderr and "HIP" not in r.stderr, r.stderr[-500:]
