"""parl_amd._torch_ops must be built from the sources in the tree: it calls the library by the signatures of its header.  CPU only."""
import os
import sys

from conftest import ROOT


def test_torch_ops_match_the_sources():
    from parl_amd import _native
    if not os.path.exists(os.path.join(ROOT, 'parl_amd', '_torch_ops.so')):
        import __graft_entry__
        __graft_entry__.build()
    csrc = os.path.join(ROOT, 'parl_amd', 'csrc')
    sys.path.insert(0, csrc)
    try:
        import srchash
    finally:
        sys.path.remove(csrc)
    assert _native.torch_ops().source_hash() == srchash.source_hash(srchash.torch_ops_files()), \
        '_torch_ops.so is stale: run python __graft_entry__.py'
