"""Which operators a status is said to come from."""
import pytest

from compiler import runtime


@pytest.mark.parametrize("status,ops", [(6, ("gemm_epilogue", "paged_attention")), (9, ("rope_append", "paged_attention"))])
def test_a_status_names_every_operator_that_reports_it(monkeypatch, status, ops):
    monkeypatch.setattr(runtime, "gemm_status", lambda device, reset: status)
    with pytest.raises(RuntimeError, match=f"status {status}") as e:
        runtime.check_status()
    assert all(f"{op} " in str(e.value) or f"{op}," in str(e.value) for op in ops)
