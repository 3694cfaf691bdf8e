"""What a call of the paged cache writes may overlap nothing that it reads: refusals of
the C entry points, without a GPU (nothing is launched)."""
import pytest

from tests.test_paged import INV, PTR, refused, rotated

QUERIES = PTR + (6 << 24)


@pytest.mark.parametrize("rows", ["k", "v"])
@pytest.mark.parametrize("heads", [1, 2, 3])
def test_append_refuses_keys_that_are_heads_of_queries_rotated_in_place(rows, heads):
    """Queries rotated where they are, and keys or values that are some of their heads:
    whether they are read before or after the rotation would be left to chance."""
    a = rotated(q_out=QUERIES)
    at = QUERIES + heads * 64 * 2
    a.k_sb, a.k_st, a.k_sh = a.q_sb, a.q_st, a.q_sh
    a.v_sb, a.v_st, a.v_sh = a.q_sb, a.q_st, a.q_sh
    setattr(a, rows, at)
    refused("nkv_paged_append", a, INV, b"q_out overlaps the rows")
