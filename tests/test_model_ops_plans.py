"""What the operators of the model plan on the host, as their workspaces show it (CPU)."""


def test_bins_of_the_table_gradient():
    """256 bins of up to 1024 ids each: with as many the parts are sorted first, in a place of their own; beyond there are more bins and
    no parts."""
    from dion_amd import _lib

    need = _lib.load().dion_amd_embedding_grad_workspace_bytes
    count, dim = 30000, 1
    parts = need(count, 262143, dim) - 262144 * 8     # (bins * rows of the index are whole)
    assert parts > count * (8 + 8)                    # the list, and the sorted parts
    assert need(count, 262144, dim) - 262144 * 8 == parts
    assert need(count, 262145, dim) - 262656 * 8 < parts
