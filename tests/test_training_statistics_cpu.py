"""CPU: the command line and the log of the step's optional statistics."""
import pytest


@pytest.mark.parametrize('args', [['--label-top', '65'], ['--label-top', '-1'], ['-K', '8', '--label-top', '9']], ids=' '.join)
def test_command_line_refuses_more_alternatives_than_there_are(args, capsys):
    import train
    with pytest.raises(SystemExit):
        train.parse(['--gan-type', 'StyleGAN2'] + args)
    assert '--label-top' in capsys.readouterr().err
    assert train.parse(['--gan-type', 'StyleGAN2', '-K', '8', '--label-top', '8']).label_top == 8
    assert train.parse(['--gan-type', 'StyleGAN2', '--label-top', '64']).label_top == 64
