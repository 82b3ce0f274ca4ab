"""The library's set-up does not depend on the shared-prefix kernels.

What the compiler and the GPU give those kernels (registers, shared memory) cannot be
varied in a test, so the source is read: the set-up that every entry shares stores their
status, and their own entry alone returns it.
"""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def body(text, start):
    """The function whose definition begins with ``start``, up to its closing brace in column 0."""
    at = text.index(start)
    return text[at:text.index('\n}\n', at)]


def test_only_its_own_entry_returns_the_prefix_status():
    text = open(os.path.join(ROOT, 'qwen3-dspark_b200', 'csrc', 'dspark_b200.cu')).read()
    info = body(text, 'int device_info(int dev, DeviceInfo* out) {')
    assert 'prefix::' not in info and info.count('prefix_') == 2      # stored, never looked at
    assert 'd.prefix_status = prefix_setup(d.max_smem_optin);' in info
    assert len(re.findall(r'dev\.prefix_status', text)) == 2
    entry = body(text, 'int dspark_prefix_attn(')
    assert 'if (dev.prefix_status != DSPARK_OK) return dev.prefix_status;' in entry
    assert entry.index('dev.prefix_status') < entry.index('<<<')
