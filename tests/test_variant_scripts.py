"""The scripts that build variants of the library link everything that the Makefile does: a library that lacks an entry point does
not load."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def makefile():
    with open(os.path.join(ROOT, 'normalizing-flows_amd', 'csrc', 'Makefile')) as f:
        return f.read()


def objects():
    return sorted(re.search(r'^OBJS := (.*)$', makefile(), re.M).group(1).replace('.o', '').split())


@pytest.mark.parametrize('script', ['build_variant.sh', 'build_fused_variant.sh', 'build_hidden_variant.sh'])
def test_every_object_is_linked(script):
    with open(os.path.join(ROOT, 'benchmarks', script)) as f:
        text = f.read()
    if script == 'build_variant.sh':
        lists = re.findall(r'^for f in ([\w ]+); do (.*)$', text, re.M)
        names = ' '.join(n for n, _ in lists).split()
        # (compiled with the Makefile's own choice of contraction)
        off = re.findall(r'^(\w+)\.o:.*\n\t.*-ffp-contract=off', makefile(), re.M)
        assert sorted(n for ns, how in lists if '-ffp-contract=off' in how for n in ns.split()) == sorted(off)
    else:
        names = re.findall(r'/(nf_\w+)\.o', text[text.index('-shared'):])
    assert sorted(names) == objects()
