"""The paged ops' decoders and host checks under AddressSanitizer and UndefinedBehaviorSanitizer, on the CPU."""

from test_host_sanitizer import _run, _san_env


def test_paged_host_tests_pass_under_asan_and_ubsan():
    res = _run(["-m", "pytest", "-q", "-x", "-p", "no:cacheprovider", "tests/test_paged_host.py"], _san_env())
    out = res.stdout + res.stderr
    assert res.returncode == 0, out[-4000:]
    assert "ERROR: AddressSanitizer" not in out and "runtime error:" not in out
    assert " passed" in out
