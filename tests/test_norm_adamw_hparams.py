"""enable_LN of the hyper-parameters: true or false and nothing that would pass for one of them (runs without a GPU)."""
import pytest

from recommenders_amd.models.deeprec import deeprec_utils as U
from recommenders_amd.models.deeprec.models._engine import dense_param_shapes, layer_norm_on

BASE = dict(model_type="xDeepFM", data_format="ffm", FEATURE_COUNT=100, FIELD_COUNT=5, dim=4, layer_sizes=[6, 7],
            activation=["relu", "relu"], dropout=[0.0, 0.0], use_DNN_part=True)


@pytest.mark.parametrize("value", [1, 0, "true", "True", 1.0, [True]])
def test_enable_ln_that_is_no_truth_value_is_refused(value):
    """A yaml file's `enable_LN: 1` trained without a norm and said nothing."""
    with pytest.raises(TypeError, match="enable_LN must be bool"):
        U.prepare_hparams(None, enable_LN=value, **BASE)
    with pytest.raises(TypeError, match="enable_LN must be bool"):  # past prepare_hparams' checks
        layer_norm_on(U.create_hparams(dict(BASE, enable_LN=value)))


def test_enable_ln_true_false_and_absent(tmp_path):
    for text, on in (("true", True), ("false", False), (None, False)):
        y = tmp_path / "hparams.yaml"
        y.write_text("model:\n  use_DNN_part: true\n" + ("  enable_LN: %s\n" % text if text else ""))
        hp = U.prepare_hparams(str(y), **{k: v for k, v in BASE.items() if k != "use_DNN_part"})
        assert layer_norm_on(hp) is on
        names = set(dense_param_shapes(hp))
        assert ({"ln_dnn_g_0", "ln_dnn_o_0", "ln_dnn_g_1", "ln_dnn_o_1"} <= names) is on
