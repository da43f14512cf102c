"""The paged key-value cache operators at the ends of what their documentation
allows: the largest tables, scores and weights at the ends of their types'
ranges, work on several streams, captured runs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32

MAX_CAPACITY = 2 ** 31 - 65537  # tokens a block table may name


def _wide_table():
    """A block table of one sequence, pages of one token, as wide as allowed (8.6 GB): page 0 throughout."""
    return torch.zeros(1, MAX_CAPACITY, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("D", [8, 5])
def test_append_at_the_end_of_the_widest_table(attn, D):
    # one new token where 131072 are offered: the pages of the others would lie behind position 2^31
    S = 131072
    table = _wide_table()
    table[0, -S:] = torch.arange(1, S + 1, dtype=torch.int32, device="cuda")
    lens = torch.tensor([MAX_CAPACITY], dtype=torch.int32, device="cuda")
    new = torch.ones(1, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(1, 1, S, D, device="cuda").to(F16) for _ in range(2))
    kc, vc = (torch.zeros(S + 2, 1, 1, D, dtype=F16, device="cuda") for _ in range(2))
    attn.kv_append(k, v, kc, vc, table, lens, new_lens=new)
    for c, x in ((kc, k), (vc, v)):
        assert torch.equal(c[S, 0, 0], x[0, 0, 0])
        assert (c[:S] == 0).all() and (c[S + 1] == 0).all()
    attn.kv_append(k, v, kc, vc, table, lens)  # all of them new
    for c, x in ((kc, k), (vc, v)):
        assert torch.equal(c[1:S + 1, 0, 0], x[0, 0])
        assert (c[0] == 0).all() and (c[S + 1] == 0).all()
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("width", [4, 5000])
def test_select_of_the_longest_list(attn, width):
    # the list's length is the largest int: the pages there are, and -1 to its end
    top = 2 ** 31 - 1
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    lens = torch.tensor([3 * 16], dtype=torch.int32, device="cuda")
    bounds = torch.zeros(1, 1, 2, 8, dtype=F16, device="cuda")
    q = torch.ones(1, 1, 1, 8, dtype=F16, device="cuda")
    pages = attn.kv_select_pages(q, bounds, table, lens, 16, top)
    assert pages.shape == (1, 1, top)
    assert pages[0, 0, :4].tolist() == [0, 1, 2, -1]
    assert int(pages[0, 0, 3:].max()) == -1 and int(pages[0, 0, 3:].min()) == -1
    assert attn.check_status(0) == 0


@pytest.mark.parametrize("lens", [[5000], [MAX_CAPACITY], [MAX_CAPACITY, 40, MAX_CAPACITY - 3]], ids=str)
def test_select_from_the_widest_table(attn, lens):
    # pages of one token; scores 0 but for a few pages up to the end (8 bytes of scratch memory a table entry)
    B, D = len(lens), 8
    table = _wide_table().expand(B, -1)
    places = [3, 17, 4990, 10 ** 9, MAX_CAPACITY - 40, MAX_CAPACITY - 5]
    table[0, places] = torch.arange(1, len(places) + 1, dtype=torch.int32, device="cuda")
    bounds = torch.zeros(len(places) + 1, 1, 2, D, dtype=F16, device="cuda")
    bounds[1:, 0, 1] = 1
    q = torch.ones(B, 1, 1, D, dtype=F16, device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pages = attn.kv_select_pages(q, bounds, table, n, 1, 8)
    for b, length in enumerate(lens):
        best = [p for p in places if p < length - 1]
        rest = [p for p in range(20) if p not in best][:7 - len(best)]  # ties to the lower page
        assert pages[b, 0].tolist() == sorted(best + rest) + [length - 1]
    assert attn.check_status(0) == 0
