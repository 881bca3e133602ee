"""What the guides tell a host to call."""
import glob
import os
import re

from aljabr_b200 import native


def test_the_documented_workspace_serves_every_call():
    """The guides' call for the largest workspace, as written there, is accepted and covers every tree."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    size = native.lib().aljabr_blackwell_kv4_tree_attention_workspace_size
    told = [m for path in sorted(glob.glob(os.path.join(root, "*.md"))) for m in
            re.findall(r"kv4TreeAttentionWorkspaceSize\(([^)]*headDim)\)", open(path, encoding="utf-8").read())]
    assert told
    for args in told:
        for heads in (1, 8):
            for D in (64, 128, 256):
                most = size(*(eval(a, {"kvHeads": heads, "headDim": D}) for a in args.split(",")))
                assert most > 0
                assert all(size(n, heads * g, heads, D) <= most for n in (1, 7, 33, 128, 256) for g in (1, 3, 4, 1024 // n) if n * g <= 1024)
