"""Every reader of a group-norm checkpoint knows the group count: GroupNorm's parameters have the
same shapes at any count, so a wrong one would load without a word and compute something else.
It is recorded beside the state ("norm_groups"), given by the caller, or the load is refused."""
import pytest
import torch


@pytest.fixture()
def paths(tmp_path):
    import ugpg
    state = ugpg.PGUNet1(3, 1, norm="group", groups=8).state_dict()
    out = {"bare": state, "unsaid": {"model_state_dict": state, "stage": 1},
           "says8": {"model_state_dict": state, "stage": 1, "norm_groups": 8},
           "batch": {"model_state_dict": ugpg.PGUNet1(3, 1).state_dict(), "stage": 1}}
    for k, v in out.items():
        torch.save(v, tmp_path / f"{k}.pth")
        out[k] = str(tmp_path / f"{k}.pth")
    return out


def readers():
    import ugpg
    from ugpg.herlev import HerlevClassificationModel, HerlevTrainer

    def trainer(path, groups):
        tr = ugpg.UncertaintyGuidedProgressiveTrainer(3, 1, device="cpu", norm="group", norm_groups=groups)
        tr.load_stage_weights(1, path)
        return tr.models[1]

    def classifier(path, groups):
        return HerlevClassificationModel(1, 7, path, norm="group", norm_groups=groups).unet

    def herlev_trainer(path, groups):
        cfg = {"device": "cpu", "epochs_per_stage": 1, "num_classes": 7, "pretrained_unet_paths": {1: path},
               "norm": "group"}
        if groups is not None:
            cfg["norm_groups"] = groups
        return HerlevTrainer(cfg).models[1].unet
    return dict(trainer=trainer, classifier=classifier, herlev_trainer=herlev_trainer)


@pytest.mark.parametrize("reader", ["trainer", "classifier", "herlev_trainer"])
def test_group_count_agrees_or_the_load_is_refused(paths, reader):
    load = readers()[reader]
    for name, groups in (("says8", 8), ("unsaid", 8), ("bare", 8)):
        assert load(paths[name], groups).inc.conv.conv_op[1].num_groups == 8
    # another count than the checkpoint's, asked for or by default; no count from either side
    for name, groups in (("says8", 16), ("says8", None), ("unsaid", None), ("bare", None)):
        with pytest.raises(ValueError, match="norm_groups"):
            load(paths[name], groups)
    for name in ("batch",):  # BatchNorm's states are told apart by their keys, as before
        with pytest.raises(RuntimeError, match="running_mean"):
            load(paths[name], 8)


def test_batch_norm_checkpoints_load_as_before(paths):
    import ugpg
    from ugpg.herlev import HerlevClassificationModel
    tr = ugpg.UncertaintyGuidedProgressiveTrainer(3, 1, device="cpu")
    tr.load_stage_weights(1, paths["batch"])
    HerlevClassificationModel(1, 7, paths["batch"])
    with pytest.raises(RuntimeError, match="running_mean"):
        tr.load_stage_weights(1, paths["unsaid"])
    with pytest.raises(RuntimeError, match="running_mean"):
        HerlevClassificationModel(1, 7, paths["says8"])
