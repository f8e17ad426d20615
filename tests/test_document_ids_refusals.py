"""What dgl_document_ids refuses before anything is launched (no GPU needed)."""
import pytest

from dgl_amd import _lib

FAKE = 4096                                   # never dereferenced: the checks come first


@pytest.mark.parametrize("change,word", [
    ({"B": 0}, b"B=0"), ({"Lq": -1}, b"Lq=-1"), ({"Lk": (1 << 24) + 1}, b"Lk="), ({"doc_q": None}, b"NULL"), ({"doc_k": None}, b"NULL"),
    ({"ids_q": None}, b"NULL"), ({"ids_k": None}, b"NULL"), ({"stride_k": -7}, b"stride"), ({"ws": None}, b"workspace"),
    ({"ws": FAKE + 4}, b"workspace"), ({"B": 1 << 30, "Lk": 1 << 20}, b"many"),
])
def test_document_ids_refuse(change, word):
    lib = _lib.load()
    a = dict(B=2, Lq=5, Lk=7, doc_q=FAKE, stride_q=5, doc_k=FAKE, stride_k=7, ids_q=FAKE, ids_k=FAKE, ws=FAKE, stream=None)
    a.update(change)
    assert lib.dgl_document_ids(*a.values()) == -1
    assert word in lib.dgl_last_error_string()


def test_workspace_holds_twice_the_keys():
    lib = _lib.load()
    for B, Lk in ((1, 0), (3, 1), (2, 1000), (1, 1 << 24)):
        floats = lib.dgl_document_ids_workspace_floats(B, Lk)
        assert floats >= 3 * B * 2 * Lk and floats >= 3 * B * 64
    assert lib.dgl_document_ids_workspace_floats(1, -1) == -1 and lib.dgl_document_ids_workspace_floats(0, 4) == -1
