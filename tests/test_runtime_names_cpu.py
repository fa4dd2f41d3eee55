"""soinfer.runtime names the batch cache beside the MLP drivers."""


def test_paged_kv_is_a_name_of_the_package():
    import soinfer.runtime as runtime

    assert "paged_kv" in runtime.__all__ and runtime.paged_kv.PagedKV4.__module__ == "soinfer.runtime.paged_kv"
