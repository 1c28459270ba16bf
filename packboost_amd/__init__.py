"""packboost_amd — PackBoost's pack-parallel tree growth and pack prediction on MI355X (gfx950).

Exports the reference's public API (packboost/__init__.py:3-6), the wrappers its README
advertises (README.md:19-20, 92-100), and operators to learn from choices and preferences.
"""

from .booster import PackBoost, Tree, TreeBuilder, TreeNode
from .choices import (ChoiceSets, PolicyLoss, PositionBias, PositionBuckets, PreferenceLoss, PreferencePairs,
                      choice_log_probs, choice_log_probs_backward, policy_loss, preference_loss)
from .config import PackBoostConfig
from .objectives import ChoicePreferenceObjective, Objective, PolicyObjective, PreferenceObjective
from .predictor import PackBoostPredictor, load_bundle, save_bundle
from .wrapper import PackBoostRegressor

__all__ = ["PackBoost", "PackBoostConfig", "PackBoostPredictor", "PackBoostRegressor", "Tree",
           "TreeNode", "TreeBuilder", "load_bundle", "save_bundle",
           "ChoiceSets", "PositionBias", "PositionBuckets", "PreferencePairs", "PolicyLoss", "PreferenceLoss",
           "choice_log_probs", "choice_log_probs_backward", "policy_loss", "preference_loss",
           "Objective", "PreferenceObjective", "ChoicePreferenceObjective", "PolicyObjective"]
__version__ = "0.1.0"
