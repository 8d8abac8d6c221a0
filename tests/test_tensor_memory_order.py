"""Tensor memory is handed out at run time: a block that waits for columns while their holder waits for that block hangs the GPU, with no limit on the wait.  Streams may overlap, so
the order of what a kernel does around its columns is what rules that out.  It is read from the sources here: no run could show it."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'n2d2_b200', 'csrc')
EVENTS = [('alloc', r'tcgen05\.alloc'), ('dealloc', r'tcgen05\.dealloc'), ('next', r'pdl_launch_dependents\(\)|griddepcontrol\.launch_dependents'),
          ('arrive wait', r'cluster_sync\(\)'), ('arrive', r'barrier\.cluster\.arrive'), ('wait', r'barrier\.cluster\.wait')]


def kernels():
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith(('.cu', '.cuh')):
            continue
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r'//[^\n]*', '', f.read())
        for at in re.finditer(r'__global__', text):
            brace = text.index('{', at.start())
            depth, end = 1, brace + 1
            while depth:
                depth += {'{': 1, '}': -1}.get(text[end], 0)
                end += 1
            body = text[brace:end]
            if 'tcgen05.alloc' in body:
                label = re.search(r'(\w+)\s*\((?=[^()]*(?:const|int|float|unsigned)\b)', text[at.start():brace].split('__launch_bounds__', 1)[-1].split(')', 1)[-1])
                yield f'{name}:{label.group(1) if label else at.start()}', body


KERNELS = dict(kernels())


def events(body):
    found = [(m.start(), kind) for names, pattern in EVENTS for kind in names.split() for m in re.finditer(pattern, body)]
    return [kind for _, kind in sorted(found, key=lambda e: e[0])]


def test_all_kernels_are_seen():
    assert len(KERNELS) >= 13, sorted(KERNELS)


@pytest.mark.parametrize('name', KERNELS)
def test_the_next_kernel_starts_behind_the_allocation(name):
    """A kernel that starts early holds its columns until the kernel before it has ended: if that one still waited for its own, it never would."""
    order = events(KERNELS[name])
    assert order.count('alloc') == order.count('dealloc') == 1
    assert 'next' not in order[:order.index('alloc')]


@pytest.mark.parametrize('name', KERNELS)
def test_columns_are_given_back_before_other_blocks_are_waited_for(name):
    """A block of a cluster that held its columns while it waits for a neighbour that waits for columns of another cluster closes a circle.  Pairs that share their
    tensor memory (cta_group::2) have a multiprocessor each to themselves: they ask for all of its columns and all of its shared memory."""
    body = KERNELS[name]
    if 'cta_group::2' in body:
        assert 'PAIR_SMEM = 227 * 1024 - 1024' in open(os.path.join(CSRC, name.split(':')[0])).read()
        return
    order = events(body)
    alloc, dealloc = order.index('alloc'), order.index('dealloc')
    # a wait in between is for blocks that arrived before they asked for columns
    ahead = order[:alloc].count('arrive') - order[:alloc].count('wait')
    assert order[alloc:dealloc].count('wait') <= ahead
