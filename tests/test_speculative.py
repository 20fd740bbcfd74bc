"""The drafting of the speculative example, on the host."""

from xpu_playground_b200.speculative import Tree, draft


def test_tree_sets_and_depths():
    t = Tree([7])
    a = t.add(0, 5)
    b = t.add(a, 6)
    c = t.add(0, 9)
    assert t.add(0, 5) == a and t.child(a, 6) == b and t.child(a, 9) is None
    assert t.depths() == [0, 1, 2, 1]
    assert t.sets() == [1, 0b11, 0b111, 0b1001] and c == 3


def test_bit_63_is_a_negative_number():
    t = Tree([0])
    for i in range(63):
        t.add(i, i + 1)
    assert t.sets()[63] == -1 and len(t.tokens) == 64


def test_draft_follows_the_newest_tokens_last_occurrences():
    t = draft([1, 2, 3, 1, 2, 4, 1], width=2, depth=2)
    assert t.tokens == [1, 2, 4, 3] and t.parents == [-1, 0, 1, 1]
    assert draft([5], 4, 4).tokens == [5]
    assert draft([1, 1, 1], width=0, depth=3).tokens == [1]
    many = draft([i % 2 for i in range(200)] + [0], width=100, depth=90)
    assert len(many.tokens) == 64
