"""The host side of the fusion block's layers under AddressSanitizer and UndefinedBehaviorSanitizer
(tests/native/host_asan_layers.cpp against the library's host-only sanitizer build, csrc
``host-asan-build``): plans, carving and argument checks over odd and limit sizes, types, alignments and
every subset of gradients."""
import os
import subprocess

import pytest

from test_sanitizers import ENV, PKG


def test_layers_host_side_under_asan_ubsan():
    exe = os.path.join(PKG, "otfuse", "lib", "asan", "host_asan_layers")
    if not os.path.exists(exe):
        pytest.skip("host sanitizer build missing: __graft_entry__.build() or "
                    "`make -C <pkg>/csrc host-asan-build` makes it")
    r = subprocess.run([exe], env=ENV, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    assert "host logic clean" in r.stdout
