"""The build copies the reference's files only where a checkout holds them."""
from oracle import make_ref


def test_absent_and_empty_checkouts_are_left_alone(tmp_path):
    before = make_ref.REF_DIR
    assert make_ref.make_ref(str(tmp_path / "nowhere")) is False
    assert make_ref.make_ref(str(tmp_path)) is False
    assert make_ref.REF_DIR == before
